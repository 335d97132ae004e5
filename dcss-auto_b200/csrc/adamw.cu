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

#include <type_traits>

#include "d1_common.cuh"
#include "d1_elem.cuh"
#include "d1_pdl.cuh"

namespace d1 {
namespace adamw {

constexpr int BLOCK = 128, THREADS = 256, WARPS = THREADS / 32, SMS = 148, NORM_GRID = SMS * 8;

// Below this eps (2^-63, the root of the smallest normal fp32 number) the square
// root of a subnormal v, which is taken as zero, would show.
constexpr double EPS_FLOOR = 1.0842021724855044e-19;

struct Args {
    const D1AdamWTensor *tensors;
    int ntensors;
    int nblocks;
    int tile;  // blocks that a warp takes at a time: 8, handed out, or 2 at fixed places
    void *m, *v;
    float *m_scale, *v_scale;
    double lr, log2_beta1, log2_beta2;
    double max_norm;
    float b1, c1, b2, c2, eps;
    int64_t *step;
    uint64_t seed;
    double *partials;            // the norm's sums, one for each of its blocks
    unsigned *arrived, *taken;   // blocks that are done, tiles handed out beyond the first of each warp; both left at 0
    int norm_parts;
    float *grad_norm;
};

// A warp's place in the tensor list (the same in every lane): a tensor's
// addresses, moved so that element i of all blocks is at index i.
struct Place {
    uintptr_t param, grad, copy;  // copy 0: none
    int full, rest;               // first block that is not whole, and how many elements it has
    int vectors, end;             // first block that is not whole or not aligned for vectors of four; first block past the tensor
    float keep;                   // 1 - lr decay
    int grad_shift;               // 2: fp32, 1: bf16
};

// The place of block `b`: the last tensor that starts at or before it, found by
// the whole warp (32 tensors looked at in one round trip).
__device__ __forceinline__ Place locate(const Args &a, int b) {
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
    p.full = (int)(t.first_block + t.count / BLOCK);
    p.rest = (int)(t.count % BLOCK);
    p.end = lo + 1 < a.ntensors ? (int)a.tensors[lo + 1].first_block : a.nblocks;
    p.keep = (float)(1. - a.lr * t.decay);
    const uintptr_t odd = (reinterpret_cast<uintptr_t>(t.param) & 15) | (reinterpret_cast<uintptr_t>(t.copy) & 7) |
                          (reinterpret_cast<uintptr_t>(t.grad) & ((4 << p.grad_shift) - 1));
    p.vectors = odd == 0 ? p.full : 0;
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

// Elements of block b from the lane's first on, up to four (b lies in the place's tensor).
__device__ __forceinline__ int left_at(const Place &p, int b) {
    return b < p.full ? 4 : imin(p.rest - 4 * (int)(threadIdx.x & 31), 4);
}
// Whether blocks b and b + 1 are whole and aligned (b or an earlier block lies in the place's tensor).
__device__ __forceinline__ bool pair_at(const Place &p, int b) { return b + 2 <= p.vectors; }

// The gradients' squares, NB blocks a warp at a time: two where a warp has few (latency
// is the bound: the clipped step of the conv policy 16.6 us, 17.9 with four), four where
// it has eight or more (memory is: 64 Mi fp32 gradients, the clipped step 387 and 333 us).
template <int NB> __global__ void __launch_bounds__(THREADS) norm_kernel(Args a) {
    __shared__ double part[WARPS];
    pdl_launch();
    const int lane = threadIdx.x & 31;
    double s = 0.;
    // a fixed share of the blocks, for a fixed order of the sum
    const int lo = (int)((int64_t)a.nblocks * blockIdx.x / gridDim.x), hi = (int)((int64_t)a.nblocks * (blockIdx.x + 1) / gridDim.x);
    Place t;
    t.end = 0;
    for (int b = lo + NB * (threadIdx.x >> 5); b < hi; b += NB * WARPS) {
        float g[NB][4] = {};
        if (b >= t.end) t = locate(a, b);
        if (b + NB <= hi && b + NB <= t.vectors)
#pragma unroll
            for (int k = 0; k < NB; k++) load_grad<true>(t, (int64_t)(b + k) * BLOCK + 4 * lane, 4, g[k]);
        else
#pragma unroll
            for (int k = 0; k < NB; k++) {
                if (b + k >= hi) break;
                if (b + k >= t.end) t = locate(a, b + k);
                load_grad<false>(t, (int64_t)(b + k) * BLOCK + 4 * lane, left_at(t, b + k), g[k]);
            }
#pragma unroll
        for (int p = 0; p < NB; p += 2) {
            float q = 0.f;
#pragma unroll
            for (int k = p; k < p + 2; k++) q += (g[k][0] * g[k][0] + g[k][1] * g[k][1]) + (g[k][2] * g[k][2] + g[k][3] * g[k][3]);
            if (!(q <= 3.402823466e38f)) {  // past fp32, from 1.8e19 on (or not finite): in 64 bits
#pragma unroll
                for (int i = 0; i < 8; i++) s += (double)g[p + i / 4][i % 4] * g[p + i / 4][i % 4];
            } else
                s += q;
        }
    }
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

__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
__device__ __forceinline__ float sqrt_approx(float x) {
    float y;
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Four codes as numbers (exact: both formats are within fp16), before their scale.
template <bool E4M3> __device__ __forceinline__ void decode4(uint32_t codes, float2 (&x)[2]) {
#pragma unroll
    for (int h = 0; h < 2; h++)
        x[h] = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes >> (16 * h)), E4M3 ? __NV_E4M3 : __NV_E5M2)));
}

// A block's scale is 2^(E - FIELD), with E the exponent of its largest
// magnitude (not below -100). A magnitude times 2^(FIELD - E + BIAS - 127) is an
// fp32 number whose bits from position 23 - mantissa on are its 8-bit code: it
// is held at the exponents where both formats have the same field, subnormal
// where the code is. `top`: the largest magnitude's bits; factor 2 is 1 unless
// the first alone would not be a normal number.
template <int FIELD, int BIAS> struct Scale {
    float first, second, scale;
    __device__ __forceinline__ explicit Scale(uint32_t top) {
        const int e = imax((int)(top & 0x7f800000u), 27 << 23);  // E + 127, in place
        const int bits = ((FIELD + BIAS + 127) << 23) - e;
        first = __int_as_float(bits);
        second = 1.f;
        scale = __int_as_float(e - (FIELD << 23));
        if (bits < 1 << 23) {
            const bool bad = top >= 0x7f800000u;  // an infinity or a NaN in the block
            first = bad ? 0.f : __int_as_float(((FIELD + 127) << 23) - e + (127 << 23));
            second = __int_as_float(BIAS << 23);
            if (bad) scale = __int_as_float(0x7fc00000);
        }
    }
};

struct Step {
    float clip, rate, inv_bc2, eps, b1, c1, b2, c2;
    uint64_t key;
};

// One block of 128, four elements a lane; the gradient as it is stored.
template <int BITS> struct Held {
    float4 p;
    uint4 g;
    typename std::conditional<BITS == 32, float4, uint32_t>::type m, v;
    float ms, vs;
};

__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// a b + c d in two columns. For 8-bit moments each operation is rounded by
// itself, so that a code is that of the formula wherever it is computed: the
// assembler joins a two-wide product and sum to a fused operation, whatever is
// asked for, so the sums are single ones.
template <int BITS> __device__ __forceinline__ float2 blend(float2 a, float b, float2 c, float d) {
    if constexpr (BITS == 32) return __ffma2_rn(a, both(b), __fmul2_rn(c, both(d)));
    const float2 p = __fmul2_rn(a, both(b)), q = __fmul2_rn(c, both(d));
    return make_float2(__fadd_rn(p.x, q.x), __fadd_rn(p.y, q.y));
}

// The step of one block, stored where its elements belong. at: the lane's first element.
template <int BITS, bool WIDE>
__device__ __forceinline__ void step_block(const Args &a, const Step &s, const Place &t, int b, const Held<BITS> &h) {
    const int lane = threadIdx.x & 31;
    const int64_t at = (int64_t)b * BLOCK + 4 * lane;
    const int left = WIDE ? 4 : left_at(t, b);
    float2 m[2], v[2];
    if constexpr (BITS == 32) {
        m[0] = make_float2(h.m.x, h.m.y), m[1] = make_float2(h.m.z, h.m.w);
        v[0] = make_float2(h.v.x, h.v.y), v[1] = make_float2(h.v.z, h.v.w);
    } else {
        decode4<true>(h.m, m);
        decode4<false>(h.v, v);
#pragma unroll
        for (int k = 0; k < 2; k++) m[k] = __fmul2_rn(m[k], both(h.ms)), v[k] = __fmul2_rn(v[k], both(h.vs));
    }
    float2 g2[2];
    if (t.grad_shift == 2) {
        g2[0] = make_float2(__uint_as_float(h.g.x), __uint_as_float(h.g.y));
        g2[1] = make_float2(__uint_as_float(h.g.z), __uint_as_float(h.g.w));
    } else {
        g2[0] = make_float2(__uint_as_float(h.g.x << 16), __uint_as_float(h.g.x & 0xffff0000u));
        g2[1] = make_float2(__uint_as_float(h.g.y << 16), __uint_as_float(h.g.y & 0xffff0000u));
    }
    const float2 p2[2] = {make_float2(h.p.x, h.p.y), make_float2(h.p.z, h.p.w)};
    float p[4];
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const float2 g = __fmul2_rn(g2[k], both(s.clip)), kept = __fmul2_rn(p2[k], both(t.keep));
        m[k] = blend<BITS>(m[k], s.b1, g, s.c1);
        v[k] = blend<BITS>(v[k], s.b2, __fmul2_rn(g, g), s.c2);
        const float2 d = __ffma2_rn(make_float2(sqrt_approx(v[k].x), sqrt_approx(v[k].y)), both(s.inv_bc2), both(s.eps));
        const float2 ratio = __fmul2_rn(m[k], make_float2(rcp_approx(d.x), rcp_approx(d.y)));
        const float2 new_p = __ffma2_rn(both(-s.rate), ratio, kept);
        p[2 * k] = new_p.x;
        p[2 * k + 1] = new_p.y;
    }
    store4<float, WIDE>(reinterpret_cast<float *>(t.param) + at, left, p);
    if (t.copy) store4<__nv_bfloat16, WIDE>(reinterpret_cast<__nv_bfloat16 *>(t.copy) + at, left, p);
    if constexpr (BITS == 32) {
        *reinterpret_cast<float4 *>((float *)a.m + at) = make_float4(m[0].x, m[0].y, m[1].x, m[1].y);
        *reinterpret_cast<float4 *>((float *)a.v + at) = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
    } else {
        const float mtop = max_nan(max_nan(fabsf(m[0].x), fabsf(m[0].y)), max_nan(fabsf(m[1].x), fabsf(m[1].y)));
        const float vtop = max_nan(max_nan(v[0].x, v[0].y), max_nan(v[1].x, v[1].y));
        const Scale<7, 7> sm(__reduce_max_sync(FULL, __float_as_uint(mtop)));
        const Scale<14, 15> sv(__reduce_max_sync(FULL, __float_as_uint(vtop)));
        const uint64_t word = mix64(s.key + ((uint64_t)b * 32 + lane));
        float ym[4], yv[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            ym[k] = __fmul_rn(fabsf(k & 1 ? m[k / 2].y : m[k / 2].x), sm.first);
            yv[k] = __fmul_rn(k & 1 ? v[k / 2].y : v[k / 2].x, sv.first);
        }
        if (sm.second != 1.f || sv.second != 1.f) {
#pragma unroll
            for (int k = 0; k < 4; k++) ym[k] = __fmul_rn(ym[k], sm.second), yv[k] = __fmul_rn(yv[k], sv.second);
        }
        uint32_t mc[4], vc[4];  // the codes in the top byte
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const uint32_t w = k < 2 ? (uint32_t)word : (uint32_t)(word >> 32);
            const uint32_t d = 2 * (k & 1 ? w >> 16 : w & 0xffffu) + 1;  // 16 random bits and a half
            mc[k] = ((__float_as_uint(ym[k]) + 8 * d) << 4 & 0x7f000000u) | (__float_as_uint(k & 1 ? m[k / 2].y : m[k / 2].x) & 0x80000000u);
            vc[k] = (__float_as_uint(yv[k]) + 16 * d) << 3;
        }
        if (__any_sync(FULL, min(min(vc[0], vc[1]), min(vc[2], vc[3])) < 1u << 24)) {  // a code of zero: only for v = 0
#pragma unroll
            for (int k = 0; k < 4; k++)
                if ((k & 1 ? v[k / 2].y : v[k / 2].x) > 0.f) vc[k] = max(vc[k], 1u << 24);
        }
        ((uint32_t *)a.m)[at >> 2] = __byte_perm(__byte_perm(mc[0], mc[1], 0x0073), __byte_perm(mc[2], mc[3], 0x0073), 0x5410);
        ((uint32_t *)a.v)[at >> 2] = __byte_perm(__byte_perm(vc[0], vc[1], 0x0073), __byte_perm(vc[2], vc[3], 0x0073), 0x5410);
        if (lane == 0) {
            a.m_scale[b] = sm.scale;
            a.v_scale[b] = sv.scale;
        }
    }
}

template <int BITS, bool WIDE>
__device__ __forceinline__ void load_block(const Args &a, const Place &t, int b, Held<BITS> &h) {
    const int64_t at = (int64_t)b * BLOCK + 4 * (threadIdx.x & 31);
    const int left = WIDE ? 4 : left_at(t, b);
    const uintptr_t g = t.grad + (at << t.grad_shift);
    if (WIDE) {
        h.p = *(reinterpret_cast<const float4 *>(t.param) + (at >> 2));
        if (t.grad_shift == 2)
            h.g = *reinterpret_cast<const uint4 *>(g);
        else
            *reinterpret_cast<uint2 *>(&h.g) = *reinterpret_cast<const uint2 *>(g);
    } else {
        float p[4];
        load4<float, false>(reinterpret_cast<const float *>(t.param) + at, left, p);
        h.p = make_float4(p[0], p[1], p[2], p[3]);
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; k++)
            w[k] = k >= left ? 0u : t.grad_shift == 2 ? reinterpret_cast<const uint32_t *>(g)[k] : reinterpret_cast<const uint16_t *>(g)[k];
        h.g = t.grad_shift == 2 ? make_uint4(w[0], w[1], w[2], w[3]) : make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, 0u, 0u);
    }
    if constexpr (BITS == 32) {
        h.m = *reinterpret_cast<const float4 *>((const float *)a.m + at);
        h.v = *reinterpret_cast<const float4 *>((const float *)a.v + at);
    } else {
        h.m = ((const uint32_t *)a.m)[at >> 2];
        h.v = ((const uint32_t *)a.v)[at >> 2];
        h.ms = a.m_scale[b];
        h.vs = a.v_scale[b];
    }
}

// The tiles of a warp: its own number first, then the next ones that nobody has
// (asked for one tile ahead). They are handed out, not shared out, because the
// SMs differ in how fast they get at memory: 128 Mi parameters in 32 bits took
// 624 us in equal shares and 563 us so. A few thousand tiles would spend more
// time at the counter than they take, so smaller steps have fixed places.
struct Tiles {
    int block, left;  // the next pair; pairs left in the tile
    unsigned next;    // lane 0's
    __device__ __forceinline__ void ask(const Args &a) {
        left = a.tile / 2;
        if (a.tile > 2 && (threadIdx.x & 31) == 0) next = atomicAdd(a.taken, 1u);
    }
    __device__ __forceinline__ explicit Tiles(const Args &a) : next(0u) {
        block = (blockIdx.x * WARPS + (threadIdx.x >> 5)) * a.tile;
        ask(a);
    }
    __device__ __forceinline__ void advance(const Args &a) {
        block += 2;
        if (--left == 0) {
            const int warps = gridDim.x * WARPS;
            const int64_t far = a.tile > 2 ? ((int64_t)warps + __shfl_sync(FULL, next, 0)) * a.tile : block + 2 * (warps - 1);
            block = far < a.nblocks ? (int)far : a.nblocks;
            ask(a);
        }
    }
};

constexpr int PER_SM = 3;  // blocks of step_kernel

// The step, in one pass over everything. 128 Mi parameters take 561 us with 32-bit
// moments (6.7 TB/s, at a copy's rate: memory is the bound) and 403 us with 8-bit ones,
// bf16 gradients and copies (5.4 TB/s, 82 %: the bound is issue slots, 77 instructions an
// element, most of them the two codes'). Two Mi and less take 10 to 17 us, latency.
template <int BITS> __global__ void __launch_bounds__(THREADS, PER_SM) step_kernel(Args a) {
    __shared__ double part[WARPS];
    __shared__ float coef[2];
    __shared__ int64_t now;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x < 2) {  // the two bias corrections, side by side
        const int64_t n = *a.step + 1;
        const double left = 1. - exp2((double)n * (lane ? a.log2_beta2 : a.log2_beta1));
        coef[lane] = lane ? (float)(1. / sqrt(left)) : (float)(a.lr / left);
        now = n;
    }
    Tiles tiles(a);
    Place t;
    t.end = 0;
    if (tiles.block < a.nblocks) t = locate(a, tiles.block);
    Step s{1.f, 0.f, 0.f, a.eps, a.b1, a.c1, a.b2, a.c2, 0u};
    if (a.max_norm > 0.) {
        // For the norm's partial sums. What came before touches the list, the step and the counter, none of
        // which the norm's kernel writes, and which was complete before that plain launch began.
        pdl_wait();
        double d = 0.;
        for (int i = threadIdx.x; i < a.norm_parts; i += THREADS) d += a.partials[i];
#pragma unroll
        for (int o = 16; o; o >>= 1) d += __shfl_xor_sync(FULL, d, o);
        if (lane == 0) part[warp] = d;
        __syncthreads();
        d = 0.;
        for (int i = 0; i < WARPS; i++) d += part[i];
        // rounded once: with another last bit of the factor, 8-bit codes would be others
        const double norm = sqrt(d), factor = a.max_norm / (norm + 1e-6);
        s.clip = factor < 1. ? (float)factor : norm == norm ? 1.f : (float)norm;
        if (blockIdx.x == 0 && threadIdx.x == 0 && a.grad_norm) *a.grad_norm = (float)norm;
    } else
        __syncthreads();
    s.rate = coef[0];
    s.inv_bc2 = coef[1];
    s.key = mix64(mix64(a.seed) + (uint64_t)now);
    while (tiles.block < a.nblocks) {
        const int b = tiles.block;
        if (b >= t.end) t = locate(a, b);
        if (!pair_at(t, b)) {
            for (int c = b; c < a.nblocks && c < b + 2; c++) {
                Held<BITS> h;
                if (c >= t.end) t = locate(a, c);
                load_block<BITS, false>(a, t, c, h);
                step_block<BITS, false>(a, s, t, c, h);
            }
            tiles.advance(a);
            continue;
        }
        Held<BITS> h[2];
        load_block<BITS, true>(a, t, b, h[0]);
        load_block<BITS, true>(a, t, b + 1, h[1]);
        for (bool more = true; more;) {
            const int c = tiles.block;
            tiles.advance(a);
            more = pair_at(t, tiles.block);
            if constexpr (BITS == 32) {
                step_block<BITS, true>(a, s, t, c, h[0]);
                step_block<BITS, true>(a, s, t, c + 1, h[1]);
                if (more) {
                    load_block<BITS, true>(a, t, tiles.block, h[0]);
                    load_block<BITS, true>(a, t, tiles.block + 1, h[1]);
                }
            } else {  // 8 bits take long to compute: the next blocks' loads are under way meanwhile
                Held<BITS> n = h[0];
                if (more) load_block<BITS, true>(a, t, tiles.block, h[0]);
                step_block<BITS, true>(a, s, t, c, n);
                n = h[1];
                if (more) load_block<BITS, true>(a, t, tiles.block + 1, h[1]);
                step_block<BITS, true>(a, s, t, c + 1, n);
            }
        }
    }
    __syncthreads();
    // every block has read the step when the last one arrives here
    if (threadIdx.x == 0) {
        __threadfence();
        if (atomicAdd(a.arrived, 1u) == gridDim.x - 1) {
            *a.arrived = *a.taken = 0u;
            *a.step = now;
        }
    }
}

}  // namespace adamw
}  // namespace d1

extern "C" int d1_adamw_work_bytes(void) { return d1::adamw::NORM_GRID * (int)sizeof(double) + 16; }

extern "C" int d1_adamw(const D1AdamWTensor *tensors, int ntensors, int64_t nblocks, int state_bits, void *m, void *v,
                        float *m_scale, float *v_scale, double lr, double beta1, double beta2, double eps,
                        double max_norm, int64_t *step, uint64_t seed, void *work, float *grad_norm, void *stream) {
    using namespace d1::adamw;
    if (nblocks > INT32_MAX - 8) return D1_ERR_TOO_LARGE;
    if (!tensors || ntensors < 1 || nblocks < 1 || (state_bits != 32 && state_bits != 8) || !m || !v || !step ||
        !work || (state_bits == 8 && (!m_scale || !v_scale)) || !(beta1 >= 0. && beta1 < 1.) ||
        !(beta2 >= 0. && beta2 < 1.) || !(eps >= 0.) || !d1::aligned_to(16, m, v, work) ||
        !d1::aligned_to(8, tensors, step) || !d1::aligned_to(4, m_scale, v_scale, grad_norm))
        return D1_ERR_BAD_ARGUMENT;
    const int tile = nblocks >= SMS * 32 * 4 * 8 ? 8 : 2;  // 8 where that makes four tiles for each warp
    double *const partials = (double *)work;
    unsigned *const counts = (unsigned *)(partials + NORM_GRID);
    Args a{tensors, ntensors, (int)nblocks, tile, m, v, m_scale, v_scale, lr, log2(beta1), log2(beta2), max_norm,
           (float)beta1, (float)(1. - beta1), (float)beta2, (float)(1. - beta2), (float)(eps > EPS_FLOOR ? eps : EPS_FLOOR),
           step, seed, partials, counts, counts + 1, 0, grad_norm};
    const cudaStream_t s = (cudaStream_t)stream;
    const int64_t norm_want = (nblocks + 2 * WARPS - 1) / (2 * WARPS), want = (nblocks + tile * WARPS - 1) / (tile * WARPS);
    const int most = SMS * PER_SM;
    cudaLaunchAttribute attr;
    cudaLaunchConfig_t cfg = d1::pdl_config(dim3((unsigned)(want < most ? want : most)), dim3(THREADS), 0, s, &attr);
    if (a.max_norm > 0.) {
        a.norm_parts = (int)(norm_want < NORM_GRID ? norm_want : NORM_GRID);
        if (nblocks >= NORM_GRID * WARPS * 8)
            norm_kernel<4><<<a.norm_parts, THREADS, 0, s>>>(a);
        else
            norm_kernel<2><<<a.norm_parts, THREADS, 0, s>>>(a);
        if (cudaError_t e = cudaGetLastError()) return (int)e;
    } else
        cfg.numAttrs = 0;
    const auto kernel = state_bits == 32 ? step_kernel<32> : step_kernel<8>;
    return (int)cudaLaunchKernelEx(&cfg, kernel, a);
}
