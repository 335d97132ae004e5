// Layer norm over the last dimension, forward and backward (sm_100a).
//
//   mean = sum(x) / n          rstd = 1 / sqrt(sum((x - mean)^2) / n + eps)
//   xhat = (x - mean) rstd     y = xhat w + b
//   g = dy w                   dx = rstd (g - mean_j(g) - xhat mean_j(g xhat))
//   dw_j = sum_r dy xhat       db_j = sum_r dy
//
// Both passes are bound by memory. A row is read once and held in registers, P
// elements a thread, by a team of 4 to 32 lanes (short rows, joined by shuffles)
// or by a block (joined through shared memory); the variance is the mean square
// of the held x - mean, not a difference of sums. In the backward pass a thread
// owns the same columns in every row, so that the weights' gradients are sums in
// its registers; a block writes one partial sum for each column, and a second,
// small launch adds the blocks' in a fixed order.
//
// Rows are read as 16-byte vectors (VEC = 16 / size) where base, pitch and n
// allow. Else 16-bit types are taken in pairs of columns (VEC = 2; a pair at an
// odd place is two loads) and fp32 column by column (VEC = 1). A warp's columns
// are 32 P in a row, so that a thread's lie at fixed distances, and only the
// last warp has to look where the row ends.
#include "d1_elem.cuh"
#include "d1_pdl.cuh"
#include "d1_rows.h"

namespace d1 {
namespace ln {

constexpr int SMS = 148;
constexpr int HELD_FORWARD = 32768;  // longest rows held in registers

template <class T> __device__ __forceinline__ float2 pair_f32(const T *e) { return make_float2(to_f32(e[0]), to_f32(e[1])); }
template <> __device__ __forceinline__ float2 pair_f32<__nv_bfloat16>(const __nv_bfloat16 *e) {
    const uint32_t w = *reinterpret_cast<const uint32_t *>(e);
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 pair_f32<__half>(const __half *e) {
    return __half22float2(*reinterpret_cast<const __half2 *>(e));
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// Loads from and stores to shared memory by its own addresses (32 bits), so
// that none of them becomes a generic access.
template <int BYTES> struct Word;
template <> struct Word<2> {
    using U = uint16_t;
    static __device__ __forceinline__ U load(uint32_t at) {
        U v;
        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at) : "memory");
        return v;
    }
    static __device__ __forceinline__ void store(uint32_t at, U v) { asm volatile("st.shared.u16 [%0], %1;" ::"r"(at), "h"(v) : "memory"); }
};
template <> struct Word<4> {
    using U = uint32_t;
    static __device__ __forceinline__ U load(uint32_t at) {
        U v;
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
        return v;
    }
    static __device__ __forceinline__ void store(uint32_t at, U v) { asm volatile("st.shared.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory"); }
};
template <> struct Word<8> {
    using U = uint2;
    static __device__ __forceinline__ U load(uint32_t at) {
        U v;
        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
        return v;
    }
};
template <> struct Word<16> {
    using U = uint4;
    static __device__ __forceinline__ U load(uint32_t at) {
        U v;
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
        return v;
    }
    static __device__ __forceinline__ void store(uint32_t at, U v) {
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
    }
};
__device__ __forceinline__ uint32_t shared_address(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
template <class E> __device__ __forceinline__ E load_shared(uint32_t at) {
    const auto w = Word<sizeof(E)>::load(at);
    return *reinterpret_cast<const E *>(&w);
}

// A thread's columns: element k of its P is column start + (k / VEC) STEP + k % VEC.
template <int VEC, int P, int G> struct Columns {
    static constexpr int LANES = G ? G : 32, STEP = LANES * VEC;
    int start, left;  // left: columns of the row from `start` on
    bool full;        // every column of the warp is in the row
    __device__ __forceinline__ explicit Columns(int n) {
        const int warp = G ? 0 : threadIdx.x >> 5, lane = threadIdx.x % LANES;
        start = warp * 32 * P + lane * VEC;
        left = n - start;
        full = G ? n == G * P : n >= (warp + 1) * 32 * P;
    }
    static __device__ __forceinline__ int offset(int k) { return k / VEC * STEP + k % VEC; }
};

// P elements of a row in registers, as P / VEC vectors.
template <class T, int VEC, int P, int G> struct Held {
    using C = Columns<VEC, P, G>;
    Elems<T, VEC> v[P / VEC];
    // From a row in shared memory, padded with zeros.
    __device__ __forceinline__ void load_staged(uint32_t at) {
        if (VEC == 2 && (at & 3)) {
#pragma unroll
            for (int i = 0; i < P / VEC; i++) {
                v[i].v[0] = load_shared<T>(at + i * C::STEP * (int)sizeof(T));
                v[i].v[VEC - 1] = load_shared<T>(at + (i * C::STEP + 1) * (int)sizeof(T));
            }
        } else
#pragma unroll
            for (int i = 0; i < P / VEC; i++) v[i] = load_shared<Elems<T, VEC>>(at + i * C::STEP * (int)sizeof(T));
    }
    __device__ __forceinline__ void load_all(const T *at) {
        if (VEC == 2 && (reinterpret_cast<uintptr_t>(at) & 3)) {
#pragma unroll
            for (int i = 0; i < P / VEC; i++) {
                v[i].v[0] = at[i * C::STEP];
                v[i].v[VEC - 1] = at[i * C::STEP + 1];
            }
        } else
#pragma unroll
            for (int i = 0; i < P / VEC; i++) v[i] = *reinterpret_cast<const Elems<T, VEC> *>(at + i * C::STEP);
    }
    // From a row in global memory; zeros past its end.
    __device__ __forceinline__ void load(const T *at, const C &c) {
        if (c.full) {
            load_all(at);
            return;
        }
#pragma unroll
        for (int i = 0; i < P / VEC; i++) {
            const int left = c.left - i * C::STEP;
            if (VEC > 2 && left > 0) {
                v[i] = *reinterpret_cast<const Elems<T, VEC> *>(at + i * C::STEP);
            } else
#pragma unroll
                for (int e = 0; e < VEC; e++) v[i].v[e] = VEC <= 2 && e < left ? at[i * C::STEP + e] : from_f32<T>(0.f);
        }
    }
    // Elements 2k and 2k + 1 of the P.
    __device__ __forceinline__ float2 pair(int k) const {
        if constexpr (VEC == 1)
            return make_float2(to_f32(v[2 * k].v[0]), to_f32(v[2 * k + 1].v[0]));
        else
            return pair_f32<T>(&v[2 * k / VEC].v[2 * k % VEC]);
    }
};
template <class T, int VEC, int P, int G>
__device__ __forceinline__ void store_row(T *at, const Columns<VEC, P, G> &c, const float2 (&y)[P / 2]) {
    constexpr int STEP = Columns<VEC, P, G>::STEP;
    Elems<T, VEC> o[P / VEC];
#pragma unroll
    for (int k = 0; k < P; k++) o[k / VEC].v[k % VEC] = from_f32<T>(k & 1 ? y[k / 2].y : y[k / 2].x);
    if (VEC == 2 && (reinterpret_cast<uintptr_t>(at) & 3)) {
#pragma unroll
        for (int k = 0; k < P; k++)
            if (c.full || k / VEC * STEP + k % VEC < c.left) at[k / VEC * STEP + k % VEC] = o[k / VEC].v[k % VEC];
    } else if (c.full) {
#pragma unroll
        for (int i = 0; i < P / VEC; i++) *reinterpret_cast<Elems<T, VEC> *>(at + i * STEP) = o[i];
    } else
#pragma unroll
        for (int i = 0; i < P / VEC; i++) {
            if (i * STEP + VEC <= c.left)
                *reinterpret_cast<Elems<T, VEC> *>(at + i * STEP) = o[i];
            else if (VEC == 2 && i * STEP < c.left)
                at[i * STEP] = o[i].v[0];
        }
}
// The columns' weights from global memory, `other` where there are none, 0 past the row.
template <int VEC, int P, int G>
__device__ __forceinline__ void load_weights(const float *w, const Columns<VEC, P, G> &c, float other, float2 (&x)[P / 2]) {
#pragma unroll
    for (int k = 0; k < P; k++) {
        const int o = Columns<VEC, P, G>::offset(k);
        const float v = o < c.left ? w ? __ldg(w + c.start + o) : other : 0.f;
        if (k & 1)
            x[k / 2].y = v;
        else
            x[k / 2].x = v;
    }
}

// Weights in shared memory, zeros past the row: padded, and for vectors of eight
// with the halves apart, so that a warp's loads of four have no bank conflicts
// (eight in a row had eightfold ones).
template <int VEC, int P> struct SharedWeights {
    static __host__ __device__ constexpr int floats(int warps) { return warps * 32 * P; }
    static __device__ __forceinline__ int place(int j, int total) {
        return VEC == 8 ? (j & 4 ? total / 2 : 0) + j / 8 * 4 + j % 4 : j;
    }
    static __device__ __forceinline__ void fill(float *s, const float *w, float other, int n, int total) {
        for (int j = threadIdx.x; j < total; j += blockDim.x) s[place(j, total)] = j < n ? w ? __ldg(w + j) : other : 0.f;
    }
    // Elements 4q .. 4q + 3 of the thread's P.
    static __device__ __forceinline__ float4 four(const float *s, int start, int q, int total) {
        constexpr int STEP = 32 * VEC;
        if constexpr (VEC == 8)
            return *reinterpret_cast<const float4 *>(s + (q & 1 ? total / 2 : 0) + start / 2 + q / 2 * (STEP / 2));
        else if constexpr (VEC == 2) {
            const float2 a = *reinterpret_cast<const float2 *>(s + start + 2 * q * STEP), b = *reinterpret_cast<const float2 *>(s + start + (2 * q + 1) * STEP);
            return make_float4(a.x, a.y, b.x, b.y);
        } else
            return make_float4(s[start + 4 * q * STEP], s[start + (4 * q + 1) * STEP], s[start + (4 * q + 2) * STEP], s[start + (4 * q + 3) * STEP]);
    }
    static __device__ __forceinline__ float2 pair(const float *s, int start, int k, int total) {
        const float4 f = four(s, start, k / 2, total);
        return k & 1 ? make_float2(f.z, f.w) : make_float2(f.x, f.y);
    }
};

// The sum over a team of G lanes, or over the block through `part` (32 floats,
// zeros past the warps); every thread gets it. Calls in turn take turns at it.
template <int G> __device__ __forceinline__ float team_sum(float s, float *part) {
#pragma unroll
    for (int o = (G ? G : 32) / 2; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (G) return s;
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
    __syncthreads();
    float2 sum = both(0.f);
    for (int w = 0; w < (int)blockDim.x; w += 256) {  // eight warps at a time
        const float4 a = *reinterpret_cast<const float4 *>(part + w / 32), b = *reinterpret_cast<const float4 *>(part + w / 32 + 4);
        sum = __fadd2_rn(sum, __fadd2_rn(__fadd2_rn(make_float2(a.x, a.y), make_float2(a.z, a.w)), __fadd2_rn(make_float2(b.x, b.y), make_float2(b.z, b.w))));
    }
    return sum.x + sum.y;
}
// The sums of a and b: the halves of the team share the work of all steps but
// the first. part: 64 floats.
template <int G> __device__ __forceinline__ void team_sums(float &a, float &b, float *part) {
    constexpr int HALF = (G ? G : 32) / 2;
    const int lane = threadIdx.x & 31;
    const bool upper = lane & HALF;
    float s = upper ? b : a;
    s += __shfl_xor_sync(0xffffffffu, upper ? a : b, HALF);
#pragma unroll
    for (int o = HALF / 2; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (G) {
        a = __shfl_sync(0xffffffffu, s, 0, G ? G : 32);
        b = __shfl_sync(0xffffffffu, s, HALF, G ? G : 32);
        return;
    }
    if ((lane & 15) == 0) part[(threadIdx.x >> 5) * 2 + (lane >> 4)] = s;
    __syncthreads();
    float2 sum = both(0.f);
    for (int w = 0; w < (int)blockDim.x; w += 128) {  // four warps at a time
        const float4 p = *reinterpret_cast<const float4 *>(part + w / 16), q = *reinterpret_cast<const float4 *>(part + w / 16 + 4);
        sum = __fadd2_rn(sum, __fadd2_rn(__fadd2_rn(make_float2(p.x, p.y), make_float2(p.z, p.w)), __fadd2_rn(make_float2(q.x, q.y), make_float2(q.z, q.w))));
    }
    a = sum.x;
    b = sum.y;
}

// The sum of (x - mu)^2 over the columns that are in the row.
template <class T, int VEC, int P, int G>
__device__ __forceinline__ float square_sum(const Held<T, VEC, P, G> &h, const Columns<VEC, P, G> &c, float mu) {
    float2 s = both(0.f);
    if (c.full) {
#pragma unroll
        for (int k = 0; k < P / 2; k++) {
            const float2 d = __fadd2_rn(h.pair(k), both(-mu));
            s = __ffma2_rn(d, d, s);
        }
    } else {
#pragma unroll
        for (int k = 0; k < P / 2; k++) {
            const float2 d = __fadd2_rn(h.pair(k), both(-mu));
            if (Columns<VEC, P, G>::offset(2 * k) < c.left) s.x = fmaf(d.x, d.x, s.x);
            if (Columns<VEC, P, G>::offset(2 * k + 1) < c.left) s.y = fmaf(d.y, d.y, s.y);
        }
    }
    return s.x + s.y;
}
template <class T, int VEC, int P, int G> __device__ __forceinline__ float plain_sum(const Held<T, VEC, P, G> &h) {
    float2 s = both(0.f);  // elements past the row are zeros
#pragma unroll
    for (int k = 0; k < P / 2; k++) s = __fadd2_rn(s, h.pair(k));
    return s.x + s.y;
}

// Forward, R rows at a time by each team of G lanes (or the block), once. The
// rows' loads are issued together and their sums joined together; blocks are
// many and small, so that others load while one adds. 65,536 rows of 512 in bf16
// take 27 us (4.9 TB/s, 75 % of a copy's rate), 4,096 rows of 8,192 in fp32 47 us
// (87 %); what is lost is memory latency where blocks begin and end and, in 16
// bits, the joins of each row. From 2,048 columns on the 16-bit kernels hold 64 elements
// a thread under bounds that leave them 64 registers, and spill, those of fp16 most
// (up to 136 bytes stored and 312 loaded by a thread): 16,357 rows of 4,096 take 56 us
// in bf16 and 69 in fp16, 4,089 of 16,384 62 and 80.
template <class T, int VEC, int P, int G, int R>
__global__ void __launch_bounds__(G ? 256 : P == 64 ? 512 : 1024, G == 32 && P == 16 ? 4 : P == 64 ? 2 : 1)
    forward_kernel(const T *x, int64_t ldx, int64_t rows, int n, const float *__restrict__ w,
                   const float *__restrict__ b, float eps, T *y, int64_t ldy, float *__restrict__ mean,
                   float *__restrict__ rstd) {
    __shared__ __align__(16) float part[2][R][32];
    const Columns<VEC, P, G> c(n);
    constexpr int STEP = Columns<VEC, P, G>::STEP;
    if (!G) {
        for (int i = threadIdx.x; i < 2 * R * 32; i += blockDim.x) (&part[0][0][0])[i] = 0.f;
        __syncthreads();
    }
    const int64_t first = G ? ((int64_t)blockIdx.x * (256 / (G ? G : 1)) + threadIdx.x / (G ? G : 1)) * R : (int64_t)blockIdx.x * R;
    const float inv_n = 1.f / n;
    Held<T, VEC, P, G> h[R];
#pragma unroll
    for (int q = 0; q < R; q++) {
        const int64_t r = first + q < rows ? first + q : rows - 1;  // past the end: the last row again, not stored
        h[q].load(x + r * ldx + c.start, c);
    }
    float mu[R], rs[R];
#pragma unroll
    for (int q = 0; q < R; q++) mu[q] = team_sum<G>(plain_sum(h[q]), part[0][q]) * inv_n;
#pragma unroll
    for (int q = 0; q < R; q++) rs[q] = 1.f / sqrtf(team_sum<G>(square_sum(h[q], c, mu[q]), part[1][q]) * inv_n + eps);
#pragma unroll
    for (int i = 0; i < P / VEC; i++) {  // vector by vector, for few registers
        const int left = c.left - i * STEP, j = c.start + i * STEP;
        if (left <= 0) break;
        float wv[VEC], bv[VEC];
        if constexpr (VEC % 4 == 0) {
#pragma unroll
            for (int e = 0; e < VEC; e += 4) {
                *reinterpret_cast<float4 *>(wv + e) = w ? __ldg(reinterpret_cast<const float4 *>(w + j + e)) : make_float4(1.f, 1.f, 1.f, 1.f);
                *reinterpret_cast<float4 *>(bv + e) = b ? __ldg(reinterpret_cast<const float4 *>(b + j + e)) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
        } else {
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                wv[e] = w && e < left ? __ldg(w + j + e) : 1.f;
                bv[e] = b && e < left ? __ldg(b + j + e) : 0.f;
            }
        }
#pragma unroll
        for (int q = 0; q < R; q++) {
            if (first + q >= rows) break;
            Elems<T, VEC> o;
            if constexpr (VEC > 1) {
#pragma unroll
                for (int e = 0; e < VEC; e += 2) {
                    const float2 c = __fmul2_rn(__fadd2_rn(h[q].pair((i * VEC + e) / 2), both(-mu[q])), both(rs[q]));
                    const float2 f = __ffma2_rn(c, make_float2(wv[e], wv[e + 1]), make_float2(bv[e], bv[e + 1]));
                    o.v[e] = from_f32<T>(f.x);
                    o.v[e + 1] = from_f32<T>(f.y);
                }
            } else
                o.v[0] = from_f32<T>(fmaf((to_f32(h[q].v[i].v[0]) - mu[q]) * rs[q], wv[0], bv[0]));
            T *const at = y + (first + q) * ldy + j;
            if (VEC == 2 && (left == 1 || (reinterpret_cast<uintptr_t>(at) & 3))) {
                at[0] = o.v[0];
                if (left > 1) at[1] = o.v[VEC - 1];
            } else
                *reinterpret_cast<Elems<T, VEC> *>(at) = o;
        }
    }
    if ((G ? threadIdx.x % (G ? G : 1) : threadIdx.x) == 0)
#pragma unroll
        for (int q = 0; q < R; q++)
            if (first + q < rows) {
                if (mean) mean[first + q] = mu[q];
                if (rstd) rstd[first + q] = rs[q];
            }
}

// ---------------------------------------------------------------- rows on their way through shared memory

__device__ __forceinline__ void copy_async16(uint32_t to, const void *from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
// 16 bytes, of which the first `size` are read and the others zero.
__device__ __forceinline__ void copy_async16(uint32_t to, const void *from, int size) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(size) : "memory");
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void wait_copies() { asm volatile("cp.async.wait_group %0;" ::"n"(N < 0 ? 0 : N) : "memory"); }

// A team's rows of x (row, row + step, ...) on their way to shared memory, DEPTH
// of them with the present one, each padded with zeros to the team's columns.
// Where rows are vectors (VECTOR) a thread copies what it will use itself and
// needs no barrier to see it. Else the team copies the row's 16-byte pieces,
// the row keeping its offset within 16 bytes, and a barrier makes them visible;
// the first piece then brings the end of the row before, but where that would
// reach out of the matrix the piece is copied element by element.
template <class T, int VEC, int P, int G> struct Rows {
    static constexpr bool VECTOR = VEC * sizeof(T) == 16;
    using C = Columns<VEC, P, G>;
    const T *at;  // the next row to fetch
    int64_t pitch;
    int left;  // rows
    uintptr_t origin;  // where the matrix begins
    __device__ __forceinline__ Rows(const T *x, int64_t ld, int64_t rows, int64_t row, int64_t step)
        : at(x + row * ld), pitch(step * ld), left(row < rows ? (int)((rows - row + step - 1) / step) : 0),
          origin(reinterpret_cast<uintptr_t>(x)) {}
    static __host__ __device__ constexpr int bytes(int warps) { return (G ? G : warps * 32) * P * (int)sizeof(T) + (VECTOR ? 0 : 16); }
    __device__ __forceinline__ void fetch(uint32_t stage, const C &c, int n) {
        if (left <= 0) return;
        if (VECTOR) {
            const uint32_t to = stage + c.start * (int)sizeof(T);
#pragma unroll
            for (int i = 0; i < P / VEC; i++)
                if (c.full || i * C::STEP < c.left) copy_async16(to + i * C::STEP * (int)sizeof(T), at + c.start + i * C::STEP);
        } else {
            const int threads = G ? G : blockDim.x, t = G ? threadIdx.x % (G ? G : 1) : threadIdx.x;
            const uintptr_t base = reinterpret_cast<uintptr_t>(at) & ~(uintptr_t)15;
            const int from = (int)(reinterpret_cast<uintptr_t>(at) & 15), to = from + n * (int)sizeof(T);
            // as far as a row at any offset goes, with zeros past this one's end
            for (int p = 16 * t; p < n * (int)sizeof(T) + 15; p += 16 * threads) {
                if (p < from && base < origin)
                    for (int e = from; e < 16; e += sizeof(T)) {
                        using U = typename Word<sizeof(T)>::U;
                        Word<sizeof(T)>::store(stage + e, e < to ? *reinterpret_cast<const U *>(base + e) : U(0));
                    }
                else {
                    const RowPiece piece = row_piece(reinterpret_cast<uintptr_t>(at), n * (int)sizeof(T), p);
                    copy_async16(stage + p, reinterpret_cast<const void *>(piece.from), piece.bytes);
                }
            }
        }
        left--;
        at += pitch;
    }
    // Zeros past the rows' ends in `count` places, before the first copies.
    static __device__ __forceinline__ void clear(uint32_t stage, int count, int bytes, int n) {
        const int threads = G ? G : blockDim.x, t = G ? threadIdx.x % (G ? G : 1) : threadIdx.x;
        for (int s = 0; s < count; s++)
            for (int p = n * (int)sizeof(T) / 16 * 16 + 16 * t; p < bytes; p += 16 * threads)
                Word<16>::store(stage + s * bytes + p, make_uint4(0u, 0u, 0u, 0u));
    }
    // Where the thread's first element of the row at `row` is in its place.
    static __device__ __forceinline__ uint32_t staged(uint32_t stage, const T *row, const C &c) {
        return stage + (VECTOR ? 0 : (uint32_t)(reinterpret_cast<uintptr_t>(row) & 15)) + c.start * (int)sizeof(T);
    }
};

// Forward of rows over 1,024 where forward_kernel is not faster: a block takes row
// after row, through shared memory, with the weights there too. 43,690 rows of
// 1,536 in bf16 take 55 us (74 % of a copy's rate), 60,349 of 1,112 72 us (57 %),
// 27,526 of 2,438 (no vectors) 71 us; its bound is the two joins of each row.
constexpr int LONG_DEPTH = 3;
template <class T, int VEC>
__global__ void __launch_bounds__(1024, 1)
    long_forward_kernel(const T *x, int64_t ldx, int64_t rows, int n, const float *__restrict__ w,
                        const float *__restrict__ b, float eps, T *y, int64_t ldy,
                        float *__restrict__ mean, float *__restrict__ rstd) {
    constexpr int P = 16, DEPTH = LONG_DEPTH;
    using R = Rows<T, VEC, P, 0>;
    using W = SharedWeights<VEC, P>;
    extern __shared__ __align__(16) unsigned char space[];
    __shared__ __align__(16) float part[4][32];
    const Columns<VEC, P, 0> c(n);
    const int warps = blockDim.x >> 5, bytes = R::bytes(warps), total = W::floats(warps);
    float *const sw = reinterpret_cast<float *>(space), *const sb = sw + total;
    const uint32_t ring = shared_address(space) + 8 * total;
    R::clear(ring, DEPTH, bytes, n);
    for (int i = threadIdx.x; i < 128; i += blockDim.x) (&part[0][0])[i] = 0.f;
    W::fill(sw, w, 1.f, n, total);
    W::fill(sb, b, 0.f, n, total);
    __syncthreads();
    const int64_t step = gridDim.x;
    int64_t r = blockIdx.x;
    R next(x, ldx, rows, r, step);
#pragma unroll
    for (int d = 0; d < DEPTH - 1; d++) {
        next.fetch(ring + d * bytes, c, n);
        commit_copies();
    }
    if (!R::VECTOR) {
        wait_copies<DEPTH - 2>();
        __syncthreads();
    }
    const float inv_n = 1.f / n;
    const T *row = x + r * ldx;
    T *out = y + r * ldy + c.start;
    int slot = 0, turn = 0;
    for (; r < rows; r += step) {
        if (R::VECTOR) wait_copies<DEPTH - 2>();
        Held<T, VEC, P, 0> h;
        h.load_staged(R::staged(ring + slot * bytes, row, c));
        const float mu = team_sum<0>(plain_sum(h), part[turn]) * inv_n;
        const float mine = square_sum(h, c, mu);
        // every thread has read the row before this one: its place takes the next
        next.fetch(ring + (slot == 0 ? DEPTH - 1 : slot - 1) * bytes, c, n);
        commit_copies();
        if (!R::VECTOR) wait_copies<DEPTH - 2>();
        const float rs = 1.f / sqrtf(team_sum<0>(mine, part[turn + 1]) * inv_n + eps);
        turn ^= 2;
        float2 o[P / 2];
#pragma unroll
        for (int q = 0; q < P / 4; q++) {
            const float4 w4 = W::four(sw, c.start, q, total), b4 = W::four(sb, c.start, q, total);
            o[2 * q] = __ffma2_rn(__fmul2_rn(__fadd2_rn(h.pair(2 * q), both(-mu)), both(rs)), make_float2(w4.x, w4.y), make_float2(b4.x, b4.y));
            o[2 * q + 1] = __ffma2_rn(__fmul2_rn(__fadd2_rn(h.pair(2 * q + 1), both(-mu)), both(rs)), make_float2(w4.z, w4.w), make_float2(b4.z, b4.w));
        }
        store_row<T, VEC, P, 0>(out, c, o);
        if (threadIdx.x == 0) {
            if (mean) mean[r] = mu;
            if (rstd) rstd[r] = rs;
        }
        row += step * ldx;
        out += step * ldy;
        slot = slot == DEPTH - 1 ? 0 : slot + 1;
    }
}

// dx of the rows that a team (8 to 32 lanes, or the block) takes, and the
// block's partial sums of dw and db in work[blockIdx.x]. Up to P = 16 the weights
// and dy w stay in registers; with 32 the weights are in shared memory and dy w
// is taken again. 16,384 rows of 4,096 in bf16 take 77 us (5.2 TB/s, 80 % of a
// copy's rate), 65,536 of 512 38 us (82 %), 5,577 of 12,032 103 us (60 %): a row's
// join stands between its loads and its stores. Rows that are no vectors are
// bound by instructions, a shared load and a store for each element or pair
// (60,404 of 1,111: 132 us, 47 %).
template <class T, int VEC, int P, int G, int DEPTH, int MOST>
__global__ void __launch_bounds__(MOST, P == 8 && G ? 3 : P == 8 || MOST == 256 ? 2 : 1)
    backward_kernel(const T *__restrict__ dy, int64_t lddy, const T *__restrict__ x, int64_t ldx, int64_t rows, int n,
                    const float *__restrict__ w, const float *__restrict__ mean, const float *__restrict__ rstd,
                    T *__restrict__ dx, int64_t lddx, float *__restrict__ work) {
    constexpr int TEAMS = G ? 256 / (G ? G : 1) : 1;
    using C = Columns<VEC, P, G>;
    using R = Rows<T, VEC, P, G>;
    using W = SharedWeights<VEC, P>;
    // with two places a row is waited for at its beginning, and its mean and rstd come with the row before it
    constexpr bool KEEP = P <= 16, LATE = DEPTH == 2, EARLY = R::VECTOR || LATE;
    constexpr int STATS = LATE ? 3 : DEPTH;
    extern __shared__ __align__(16) unsigned char space[];
    __shared__ __align__(16) float part[2][64];
    __shared__ float stats[TEAMS][STATS][2];  // mean and rstd of the rows on their way
    pdl_launch();
    const C c(n);
    const int warps = blockDim.x >> 5, team = G ? threadIdx.x / (G ? G : 1) : 0, bytes = R::bytes(warps), total = W::floats(warps);
    const uint32_t ring = shared_address(space) + team * (DEPTH * 2 * bytes);
    float *const sw = reinterpret_cast<float *>(space + TEAMS * DEPTH * 2 * bytes);
    R::clear(ring, 2 * DEPTH, bytes, n);
    for (int i = threadIdx.x; i < 128; i += blockDim.x) (&part[0][0])[i] = 0.f;
    if (!KEEP) W::fill(sw, w, 1.f, n, total);
    __syncthreads();
    const int64_t step = (int64_t)gridDim.x * TEAMS, first = (int64_t)blockIdx.x * TEAMS + team;
    R next_x(x, ldx, rows, first, step), next_dy(dy, lddy, rows, first, step);
    const int t = G ? threadIdx.x % (G ? G : 1) : threadIdx.x;
    const float *next_stat = (t == 0 ? mean : rstd) + first;
    const uint32_t stat_at = shared_address(&stats[team][0][0]);
    int stats_left = next_x.left;
    auto fetch_stat = [&](int place) {
        if (t < 2 && stats_left > 0) {
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(stat_at + 8 * place + 4 * t), "l"(next_stat) : "memory");
            next_stat += step;
        }
        stats_left--;
    };
    auto fetch = [&](int slot, int place) {
        fetch_stat(place);
        next_x.fetch(ring + slot * 2 * bytes, c, n);
        next_dy.fetch(ring + slot * 2 * bytes + bytes, c, n);
        commit_copies();
    };
#pragma unroll
    for (int d = 0; d < DEPTH - 1; d++) {
        if (LATE) fetch_stat(0);
        fetch(d, LATE ? 1 : d);
    }
    float2 wk[P / 2], aw[P / 2], ab[P / 2];
    if (KEEP) load_weights<VEC, P, G>(w, c, 1.f, wk);
#pragma unroll
    for (int k = 0; k < P / 2; k++) aw[k] = ab[k] = both(0.f);
    auto weight = [&](int k) { return KEEP ? wk[k] : W::pair(sw, c.start, k, total); };
    const float inv_n = 1.f / n;
    wait_copies<DEPTH - 2>();
    __syncthreads();
    float2 stat = load_shared<float2>(stat_at);
    const T *xr = x + first * ldx, *dr = dy + first * lddy;
    T *out_row = dx + first * lddx + c.start;
    int slot = 0, place = 0, turn = 0;
    const int rounds = (int)((rows - (int64_t)blockIdx.x * TEAMS + step - 1) / step);  // of the block's first team
    int64_t r = first;
    for (int round = 0; round < rounds; round++) {
        const bool live = r < rows;  // the teams of a warp stay together
        const float mu = stat.x, rs = stat.y;
        // the place of the row before this one takes the next: at once where it was the thread's
        // own, else when the team has done with it
        if (LATE && round > 0) {
            wait_copies<0>();
            if (!R::VECTOR) __syncthreads();
        }
        if (EARLY) fetch(slot == 0 ? DEPTH - 1 : slot - 1, place == 0 ? STATS - 1 : place - 1);
        const uint32_t stage = ring + slot * 2 * bytes, ds = R::staged(stage + bytes, dr, c);
        float2 xhat[P / 2], g[KEEP ? P / 2 : 1], sum1 = both(0.f), sum2 = both(0.f);
        if (TEAMS == 1 || live) {
            Held<T, VEC, P, G> xv, dv;  // zeros past the row
            xv.load_staged(R::staged(stage, xr, c));
            dv.load_staged(ds);
#pragma unroll
            for (int k = 0; k < P / 2; k++) {
                const float2 d = dv.pair(k), h = __fmul2_rn(__fadd2_rn(xv.pair(k), both(-mu)), both(rs)), gk = __fmul2_rn(d, weight(k));
                sum1 = __fadd2_rn(sum1, gk);
                sum2 = __ffma2_rn(gk, h, sum2);
                aw[k] = __ffma2_rn(d, h, aw[k]);
                ab[k] = __fadd2_rn(ab[k], d);
                xhat[k] = h;
                if (KEEP) g[KEEP ? k : 0] = gk;
            }
        }
        float s1 = sum1.x + sum1.y, s2 = sum2.x + sum2.y;
        if (!LATE) wait_copies<EARLY ? DEPTH - 2 : DEPTH - 3>();  // for the row after this one
        team_sums<G>(s1, s2, part[turn]);
        turn ^= 1;
        if (G) __syncwarp();
        if (!EARLY) fetch(slot == 0 ? DEPTH - 1 : slot - 1, place == 0 ? STATS - 1 : place - 1);
        place = place == STATS - 1 ? 0 : place + 1;
        stat = load_shared<float2>(stat_at + 8 * place);
        if ((TEAMS == 1 || live) && dx) {
            const float2 c1 = both(-rs * s1 * inv_n), c2 = both(-rs * s2 * inv_n);
            Held<T, VEC, P, G> dv;
            if (!KEEP) dv.load_staged(ds);
#pragma unroll
            for (int k = 0; k < P / 2; k++)
                xhat[k] = __ffma2_rn(xhat[k], c2, __ffma2_rn(KEEP ? g[KEEP ? k : 0] : __fmul2_rn(dv.pair(k), weight(k)), both(rs), c1));
            store_row<T, VEC, P, G>(out_row, c, xhat);
        }
        r += step;
        xr += step * ldx;
        dr += step * lddy;
        out_row += step * lddx;
        slot = slot == DEPTH - 1 ? 0 : slot + 1;
    }
    if (!work) return;
    wait_copies<0>();
    float *out = work + (int64_t)blockIdx.x * 2 * n + c.start, *joined = reinterpret_cast<float *>(space);
#pragma unroll
    for (int half = 0; half < 2; half++) {
        float2(&a)[P / 2] = half ? ab : aw;
        if (G) {  // the teams' sums, added in their order
            __syncthreads();
#pragma unroll
            for (int k = 0; k < P / 2; k++) *reinterpret_cast<float2 *>(joined + (k * 256 + threadIdx.x) * 2) = a[k];
            __syncthreads();
            if (team == 0)
#pragma unroll
                for (int k = 0; k < P / 2; k++) {
                    a[k] = both(0.f);
                    for (int q = 0; q < TEAMS; q++) a[k] = __fadd2_rn(a[k], *reinterpret_cast<float2 *>(joined + (k * 256 + q * G + threadIdx.x) * 2));
                }
        }
        if (team == 0)
#pragma unroll
            for (int k = 0; k < P; k++)
                if (C::offset(k) < c.left) out[half * n + C::offset(k)] = k & 1 ? a[k / 2].y : a[k / 2].x;
    }
}

// dw and db from the blocks' partial sums: 32 columns a block, in 32 slices of the
// parts. A launch of its own because blocks end at different times; it costs 2 to
// 3 us after the rows (5,003 rows of 1,111 in fp32: 20 us in all, of which the
// bytes take 10).
__global__ void __launch_bounds__(1024)
    reduce_kernel(const float *__restrict__ work, int parts, int n, float *__restrict__ dw, float *__restrict__ db) {
    __shared__ float sums[32][33];
    pdl_wait();
    const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
    const unsigned j = blockIdx.x * 32 + lane, columns = 2u * n;  // twice the longest row passes 31 bits
    float s = 0.f;
    if (j < columns) {
#pragma unroll 8
        for (int p = slice; p < parts; p += 32) s += work[(int64_t)p * 2 * n + j];
    }
    sums[slice][lane] = s;
    __syncthreads();
    s = warp_sum(sums[lane][slice]);  // warp `slice` adds the slices of its column
    const unsigned c = blockIdx.x * 32 + slice;
    if (lane || c >= columns) return;
    if (c < (unsigned)n) {
        if (dw) dw[c] = s;
    } else if (db)
        db[c - n] = s;
}

// ---------------------------------------------------------------- rows too long for registers

// Plain passes over the row, element by element, the second and third from L2: for
// completeness more than for speed. Columns are counted without a sign: the step past
// the end of the longest rows passes 31 bits. 1,024 rows of 65,536 in fp32 take 212 us forward
// (39 % of a copy's rate) and 348 us backward (35 %), by
// loads and stores of one element each.

constexpr int WIDE = 1024;

template <class T>
__global__ void __launch_bounds__(WIDE)
    wide_forward_kernel(const T *x, int64_t ldx, int64_t rows, int n, const float *__restrict__ w,
                        const float *__restrict__ b, float eps, T *y, int64_t ldy,
                        float *__restrict__ mean, float *__restrict__ rstd) {
    __shared__ __align__(16) float part[2][32];
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const T *xr = x + r * ldx;
        float s = 0.f;
        for (unsigned j = threadIdx.x; j < (unsigned)n; j += WIDE) s += to_f32(xr[j]);
        const float mu = team_sum<0>(s, part[0]) / n;
        s = 0.f;
        for (unsigned j = threadIdx.x; j < (unsigned)n; j += WIDE) {
            const float c = to_f32(xr[j]) - mu;
            s += c * c;
        }
        const float rs = 1.f / sqrtf(team_sum<0>(s, part[1]) / n + eps);
        for (unsigned j = threadIdx.x; j < (unsigned)n; j += WIDE)
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
    __shared__ __align__(16) float part[2][64];
    int turn = 0;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const float mu = mean[r], rs = rstd[r];
        float s1 = 0.f, s2 = 0.f;
        for (unsigned j = threadIdx.x; j < (unsigned)n; j += WIDE) {
            const float g = to_f32(dy[r * lddy + j]) * (w ? w[j] : 1.f);
            s1 += g;
            s2 += g * ((to_f32(x[r * ldx + j]) - mu) * rs);
        }
        team_sums<0>(s1, s2, part[turn]);
        turn ^= 1;
        s1 /= n;
        s2 /= n;
        for (unsigned j = threadIdx.x; j < (unsigned)n; j += WIDE) {
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
    const unsigned j = blockIdx.x * 256 + threadIdx.x;
    if (j >= (unsigned)n) return;
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

template <class T> static bool vectors_of(const void *p, int64_t ld) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld * (int64_t)sizeof(T) % 16 == 0;
}
static bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

constexpr size_t SPACE = 225 * 1024;  // shared memory of an SM that blocks can have

template <class K> static int allow_space(K kernel, size_t smem) {
    return smem > 40 * 1024 ? (int)cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) : 0;
}

template <class T, int VEC>
static int forward(const T *x, int64_t ldx, int64_t rows, int n, const float *w, const float *b, float eps, T *y,
                   int64_t ldy, float *mean, float *rstd, cudaStream_t s) {
#define D1_LN_FORWARD(P, G, R, threads)                                                                               \
    do {                                                                                                              \
        const int64_t per_block = (int64_t)R * ((G) ? 256 / ((G) ? (G) : 1) : 1), blocks = (rows + per_block - 1) / per_block; \
        if (blocks > INT32_MAX) return D1_ERR_TOO_LARGE;                                                              \
        forward_kernel<T, VEC, P, G, R><<<(int)blocks, threads, 0, s>>>(x, ldx, rows, n, w, b, eps, y, ldy, mean, rstd); \
        return (int)cudaGetLastError();                                                                               \
    } while (0)
    // Sixteen elements a lane by as few lanes as hold the row, for a row's joins cost the same whatever they join:
    // 233,016 rows of 72 in bf16 take 23 us with 8 lanes, 51 with 32; 83,886 of 200 19 us with 16, 23 with 32. Element
    // by element 8 a lane are as good, and where rows are too few for the SMs, 32 lanes have the shorter way.
    const bool many = rows >= SMS * 32;
    if constexpr (VEC == 8)
        if (n <= 64 && many) D1_LN_FORWARD(16, 4, 2, 256);
    if (n <= 64) D1_LN_FORWARD(8, 8, 2, 256);
    if constexpr (VEC > 1) {
        if (n <= 128 && many) D1_LN_FORWARD(16, 8, 2, 256);
        if (n <= 256 && many) D1_LN_FORWARD(16, 16, 2, 256);
    }
    if (n <= 256) D1_LN_FORWARD(8, 32, 2, 256);
    // (12 and 24 elements a lane leave fewer idle where the bound is instructions: 120,266 rows of 279 in bf16 49 and
    // 46 us, 64,403 of 521 in fp16 50 and 44)
    if constexpr (VEC <= 2)
        if (n <= 384) D1_LN_FORWARD(12, 32, 2, 256);
    if (n <= 512) D1_LN_FORWARD(16, 32, 2, 256);
    if constexpr (VEC == 2)
        if (n <= 768) D1_LN_FORWARD(24, 32, 1, 256);
    if (n <= 1024) D1_LN_FORWARD(32, 32, 1, 256);
    // Longer rows are a block's. Where the vectors are whole, 32 elements a thread (64 of the longest) need fewer
    // joins than 16 do, and blocks that come and go keep more rows under way than resident ones with their rows in
    // shared memory: 16,384 in bf16 63 us against 72 (4,096 rows), 4,096 57 against 59 (16,384 rows, two at a time, for
    // their weights), 3,156 in fp32 47 against 53 (10,631 rows). Of 1,112 and 1,536 in bf16 it is the other way round:
    // 74 against 72, 59 against 55, and 1,111 in fp32 (element by element) 92 against 61.
    if constexpr (VEC == 4)
        D1_LN_FORWARD(32, 0, 1, block_threads(n, 32));
    else {
        if constexpr (VEC == 8)
            if (n > 8192) D1_LN_FORWARD(64, 0, 1, block_threads(n, 64));
        if constexpr (VEC > 1)
            if (n >= (VEC == 8 ? 2048 : 4097)) D1_LN_FORWARD(32, 0, 2, block_threads(n, 32));
        const int threads = block_threads(n, 16), warps = threads / 32;
        const size_t smem = (size_t)LONG_DEPTH * Rows<T, VEC, 16, 0>::bytes(warps) + 8 * (size_t)SharedWeights<VEC, 16>::floats(warps);
        if constexpr (VEC == 1)  // the others have at most 256 threads here
            if (threads > 1024 || smem + 2048 > SPACE) D1_LN_FORWARD(32, 0, 1, block_threads(n, 32));
        const auto kernel = long_forward_kernel<T, VEC>;
        if (const int e = allow_space(kernel, smem)) return e;
        const int by_threads = 1024 / threads, by_space = (int)(SPACE / (smem + 2048));
        const int64_t full = (int64_t)SMS * (by_threads < by_space ? by_threads : by_space);
        kernel<<<(int)(rows < full ? rows : full), threads, smem, s>>>(x, ldx, rows, n, w, b, eps, y, ldy, mean, rstd);
        return (int)cudaGetLastError();
    }
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
    if (n % VEC == 0 && vectors_of<T>(x, ldx) && vectors_of<T>(y, ldy) && aligned16(w) && aligned16(b))
        return forward<T, VEC>((const T *)x, ldx, rows, n, w, b, eps, (T *)y, ldy, mean, rstd, s);
    return forward<T, sizeof(T) == 2 ? 2 : 1>((const T *)x, ldx, rows, n, w, b, eps, (T *)y, ldy, mean, rstd, s);
}

// How the backward pass runs: teams of 8, 16 or 32 lanes, or blocks (lanes = 0),
// with P elements a thread, DEPTH rows in shared memory and as many blocks as
// the SMs hold at once (more would only write more partial sums). Eight elements
// a thread for rows of 513 to 1,024 that are vectors, sixteen for others, whose
// joins cost more than the idle lanes: 85,707 rows of 783 in fp16, 160 and 123 us.
// Twelve for those of 257 to 384: 120,266 of 279 in bf16, 91 us with sixteen and 70.
// Rows of 65 to 256 have sixteen too, in 8 or 16 lanes, but for element by element:
// 131,072 of 128 in bf16 40 us in 32 lanes, 22 in 8; 83,886 of 200 30 and 25.
struct Backward {
    int lanes, p, depth, threads, grid;
    size_t smem;
};
static Backward backward_shape(int64_t rows, int n, int size, bool vector) {
    Backward o;
    const bool single = size == 4 && !vector;
    o.lanes = n <= (single ? 64 : 128) ? 8 : n <= 256 && !single ? 16 : n <= 512 ? 32 : 0;
    o.p = !single && n > 64 && n <= 256 ? 16 : n <= 256 || (vector && n > 512 && n <= 1024) ? 8 : !vector && n <= 384 ? 12 : n <= 8192 ? 16 : 32;
    o.threads = o.lanes ? 256 : block_threads(n, o.p);
    const int teams = o.lanes ? 256 / o.lanes : 1;
    const size_t pair = 2 * (size_t)((o.lanes ? o.lanes : o.threads) * o.p * size + (vector ? 0 : 16));  // a row of x and one of dy
    o.depth = o.p == 32 ? 2 : 4 * pair > 160 * 1024 ? 3 : 4;
    o.smem = o.depth * pair * teams + (o.p == 32 ? 4 * (size_t)o.threads * 32 : 0);
    if (o.lanes && o.smem < (size_t)256 * o.p * 4) o.smem = (size_t)256 * o.p * 4;  // the teams' sums, joined at the end
    const int by_threads = (o.p == 8 ? o.lanes ? 768 : 1024 : 512) / o.threads, by_space = (int)(SPACE / (o.smem + 2048));
    const int resident = by_threads < by_space ? by_threads : by_space;
    const int64_t want = (rows + teams - 1) / teams, full = (int64_t)SMS * (resident < 1 ? 1 : resident);
    o.grid = (int)(want < 1 ? 1 : want < full ? want : full);
    return o;
}
// Rows that the backward pass holds: over 8,192 elements only those of 16 bits are.
static bool held_backward(int n, int size) { return n <= 8192 || (n <= 16384 && size == 2); }
static int parts_of(int64_t rows, int n, int size, bool vector) {
    if (!held_backward(n, size)) return (int)(rows < 1 ? 1 : rows < 16 ? rows : 16);
    return backward_shape(rows, n, size, vector).grid;
}

template <class T, int VEC>
static int backward(const T *dy, int64_t lddy, const T *x, int64_t ldx, int64_t rows, int n, const float *w,
                    const float *mean, const float *rstd, T *dx, int64_t lddx, float *work, cudaStream_t s) {
    constexpr bool VECTOR = VEC * sizeof(T) == 16;
    const Backward o = backward_shape(rows, n, sizeof(T), VECTOR);
    auto kernel = backward_kernel<T, VEC, 8, 8, 4, 256>;  // lanes and p are 8
    if (o.lanes == 32)
        kernel = backward_kernel<T, VEC, 16, 32, 4, 256>;
    else if (o.lanes == 0)
        kernel = o.threads <= 256 ? backward_kernel<T, VEC, 16, 0, 4, 256> : backward_kernel<T, VEC, 16, 0, 4, 512>;
    if constexpr (VEC == 1) {
        if (o.lanes == 32 && o.p == 8) kernel = backward_kernel<T, VEC, 8, 32, 4, 256>;
    } else {
        if (o.lanes == 8 && o.p == 16) kernel = backward_kernel<T, VEC, 16, 8, 4, 256>;
        if (o.lanes == 16) kernel = backward_kernel<T, VEC, 16, 16, 4, 256>;
    }
    if constexpr (VECTOR) {
        if (o.lanes == 0 && o.p == 8) kernel = backward_kernel<T, VEC, 8, 0, 4, 512>;
    } else if (o.p == 12)
        kernel = backward_kernel<T, VEC, 12, 32, 4, 256>;
    if constexpr (sizeof(T) == 2) {
        if (o.p == 32) kernel = backward_kernel<T, VEC, 32, 0, 2, 512>;
    } else if (o.depth == 3)
        kernel = backward_kernel<T, VEC, 16, 0, 3, 512>;
    if (const int e = allow_space(kernel, o.smem)) return e;
    kernel<<<o.grid, o.threads, o.smem, s>>>(dy, lddy, x, ldx, rows, n, w, mean, rstd, dx, lddx, work);
    return (int)cudaGetLastError();
}

template <class T>
static int backward_any(const void *dy, int64_t lddy, const void *x, int64_t ldx, int64_t rows, int n, const float *w,
                        const float *mean, const float *rstd, void *dx, int64_t lddx, float *dw, float *db,
                        float *work, cudaStream_t s) {
    constexpr int VEC = 16 / sizeof(T);
    const bool sums = dw || db, vector = n % VEC == 0 && vectors_of<T>(x, ldx) && vectors_of<T>(dy, lddy) &&
                                         (!dx || vectors_of<T>(dx, lddx)) && aligned16(w);
    const int parts = parts_of(rows, n, sizeof(T), vector);
    int e = 0;
    if (!held_backward(n, sizeof(T))) {
        if (dx && rows)
            wide_rows_kernel<T><<<(int)(rows < SMS * 2 ? rows : SMS * 2), WIDE, 0, s>>>(
                (const T *)dy, lddy, (const T *)x, ldx, rows, n, w, mean, rstd, (T *)dx, lddx);
        if ((e = (int)cudaGetLastError())) return e;
        if (sums)
            wide_columns_kernel<T><<<dim3(((unsigned)n + 255) / 256, parts), 256, 0, s>>>((const T *)dy, lddy, (const T *)x, ldx,
                                                                                rows, n, mean, rstd, work);
        e = (int)cudaGetLastError();
    } else if (vector)
        e = backward<T, VEC>((const T *)dy, lddy, (const T *)x, ldx, rows, n, w, mean, rstd, (T *)dx, lddx, sums ? work : nullptr, s);
    else
        e = backward<T, sizeof(T) == 2 ? 2 : 1>((const T *)dy, lddy, (const T *)x, ldx, rows, n, w, mean, rstd, (T *)dx, lddx,
                                                sums ? work : nullptr, s);
    if (e || !sums) return e;
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = pdl_config(dim3((2u * n + 31) / 32), dim3(1024), 0, s, &attr);
    return (int)cudaLaunchKernelEx(&cfg, reduce_kernel, (const float *)work, parts, n, dw, db);
}

}  // namespace ln
}  // namespace d1

extern "C" int d1_layer_norm(const void *x, int64_t ldx, int type, int64_t rows, int n, const float *weight,
                             const float *bias, float eps, void *y, int64_t ldy, float *mean, float *rstd,
                             void *stream) {
    using namespace d1;
    if (!type_ok(type) || rows < 0 || n < 1 || (rows && (!x || !y)) || !(eps >= 0.f) || ldx < 0 || ldy < 0 ||
        (rows > 1 && ldy < n) || !element_aligned(x, type) || !element_aligned(y, type) ||
        !aligned_to(4, weight, bias, mean, rstd))
        return D1_ERR_BAD_ARGUMENT;
    if (rows == 0) return 0;
    const int64_t size = type == D1_TYPE_F32 ? 4 : 2;
    const RowSpan in{(uintptr_t)x, rows, n * size, ldx * size}, result{(uintptr_t)y, rows, n * size, ldy * size};
    if (x == y ? rows > 1 && ldx != ldy : rows_overlap(in, result)) return D1_ERR_BAD_ARGUMENT;
    const cudaStream_t s = (cudaStream_t)stream;
    if (type == D1_TYPE_F32) return ln::forward_any<float>(x, ldx, rows, n, weight, bias, eps, y, ldy, mean, rstd, s);
    if (type == D1_TYPE_BF16)
        return ln::forward_any<__nv_bfloat16>(x, ldx, rows, n, weight, bias, eps, y, ldy, mean, rstd, s);
    return ln::forward_any<__half>(x, ldx, rows, n, weight, bias, eps, y, ldy, mean, rstd, s);
}

extern "C" int d1_layer_norm_parts(int64_t rows, int n) {
    if (rows < 0 || n < 1) return D1_ERR_BAD_ARGUMENT;
    int most = 0;  // of either size of element and either alignment
    for (int k = 0; k < 4; k++) {
        const int parts = d1::ln::parts_of(rows, n, k & 1 ? 4 : 2, k & 2);
        if (parts > most) most = parts;
    }
    return most;
}

extern "C" int d1_layer_norm_backward(const void *dy, int64_t lddy, const void *x, int64_t ldx, int type, int64_t rows,
                                      int n, const float *weight, const float *mean, const float *rstd, void *dx,
                                      int64_t lddx, float *dweight, float *dbias, float *work, void *stream) {
    using namespace d1;
    if (!type_ok(type) || rows < 0 || n < 1 || (rows && (!dy || !x || !mean || !rstd)) || lddy < 0 || ldx < 0 ||
        lddx < 0 || (dx && rows > 1 && lddx < n) || ((dweight || dbias) && !work) || !element_aligned(x, type) ||
        !element_aligned(dy, type) || !element_aligned(dx, type) ||
        !aligned_to(4, weight, mean, rstd, dweight, dbias) || !aligned_to(16, work))
        return D1_ERR_BAD_ARGUMENT;
    const int64_t size = type == D1_TYPE_F32 ? 4 : 2;
    const RowSpan result{(uintptr_t)dx, dx ? rows : 0, n * size, lddx * size};
    if (rows_overlap(result, {(uintptr_t)x, rows, n * size, ldx * size}) || rows_overlap(result, {(uintptr_t)dy, rows, n * size, lddy * size}))
        return D1_ERR_BAD_ARGUMENT;
    const cudaStream_t s = (cudaStream_t)stream;
    if (type == D1_TYPE_F32)
        return ln::backward_any<float>(dy, lddy, x, ldx, rows, n, weight, mean, rstd, dx, lddx, dweight, dbias, work, s);
    if (type == D1_TYPE_BF16)
        return ln::backward_any<__nv_bfloat16>(dy, lddy, x, ldx, rows, n, weight, mean, rstd, dx, lddx, dweight, dbias,
                                               work, s);
    return ln::backward_any<__half>(dy, lddy, x, ldx, rows, n, weight, mean, rstd, dx, lddx, dweight, dbias, work, s);
}
