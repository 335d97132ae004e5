// Log-probabilities of given tokens, with the distribution's entropy and its
// likeliest alternatives, and their gradient (sm_100a).
//
// For one row of logits x over a vocabulary, with z_j = (x_j - max x) / T over
// the tokens that are not left out (legal bit clear, or logit -inf):
//
//   S = sum_j e^{z_j}     log p_j = z_j - log S     H = log S - sum_j z_j e^{z_j} / S
//   d log p_t / d x_j = (1[j = t] - p_j) / T        d H / d x_j = -p_j (log p_j + H) / T
//
// A row with nothing left has log p = -inf, H = 0, no alternatives and a zero
// gradient. A NaN or +inf that is not left out makes S, log p, H and the gradient of
// what is not left out NaN.
//
// One pass over the logits: each thread keeps a running maximum m, the sum s of
// 2^{(x - m) c} and the sum t of (x - m) c 2^{(x - m) c}, with c = log2(e) / T,
// for a batch of 16-byte vectors at a time (the two sums are scaled down once a
// batch, when the maximum has moved). The joins over threads, warps and the
// blocks of a cluster use the same rule, in a fixed order.
//
// The k alternatives need no second pass over the row. A thread's running
// maximum is the largest of the logits that it saw, so the k-th largest of the
// threads' maxima (found by bisection with counts over the warp) bounds the
// k-th largest logit from below, and only threads whose maximum reaches it saw
// a candidate: about k columns of vectors are read again, from L2 (of long
// rows, only the cells of them whose own maximum reaches it). The candidates
// (about k of them, unless logits are equal in great numbers) are ordered by
// counting, for each, how many are better. Where more of them reach the bound than
// the list holds, one more pass takes what is above the bound and the first that equal
// it (600 rows of 131,072 equal logits in bf16, k = 20: 570 us in place of 53), and only
// where hundreds are above it, or where few long rows are split over SMs, a search in
// k rounds (4 such rows: 98 us in place of 13).
#include <float.h>
#include <math_constants.h>

#include "d1_elem.cuh"
#include "d1_rows.h"

namespace d1 {
namespace lp {

constexpr int THREADS = 256, WARPS = THREADS / 32, MAX_TOP = 32, MAX_CLUSTER = 8, CAP = 768;
constexpr int SMS = 148;
constexpr int UNROLL = 4;           // vectors a thread has in flight
constexpr int SHORT_VOCAB = 64;     // rows up to here are held in the registers of 8 lanes
constexpr int MIDDLE_VOCAB = 8192;  // rows up to here are a warp's
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// A candidate as one number: the logit in whole-number order (-0 equal to +0,
// NaN above all, 0 for a token that is left out), then the lower index first.
__device__ __forceinline__ uint32_t order_key(float x) {
    if (x != x) return 0xffffffffu;
    if (x == -CUDART_INF_F) return 0u;
    const uint32_t u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t candidate(uint32_t key, int index) { return (uint64_t)key << 32 | ~(uint32_t)index; }
__device__ __forceinline__ uint32_t key_of(uint64_t c) { return (uint32_t)(c >> 32); }
__device__ __forceinline__ int index_of(uint64_t c) { return (int)~(uint32_t)c; }
__device__ __forceinline__ float logit_of(uint64_t c) {
    const uint32_t k = key_of(c);
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// Running maximum and sums; m = -inf: nothing yet.
struct Acc {
    float m, s, t;
};

__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

__device__ __forceinline__ void rescale(Acc &a, float top, float c) {
    if (!(top <= a.m)) {
        const float d = fmaxf((a.m - top) * c, -1e4f), f = ex2(d);
        a.t = f * fmaf(d, a.s, a.t);
        a.s *= f;
        a.m = top;
    }
}
__device__ __forceinline__ void add_pair(float2 &s, float2 &t, float2 x, float m, float c) {
    // below 2^-200 the term is zero; the bound also takes in -inf (and -inf - -inf)
    float2 z = __fmul2_rn(__fadd2_rn(x, both(-m)), both(c));
    z.x = fmaxf(z.x, -200.f);
    z.y = fmaxf(z.y, -200.f);
    const float2 e = make_float2(ex2(z.x), ex2(z.y));
    s = __fadd2_rn(s, e);
    t = __ffma2_rn(z, e, t);
}
// top: the largest of x (a NaN if there is one).
template <int N> __device__ __forceinline__ void take(Acc &a, const float2 (&x)[N], float top, float c) {
    rescale(a, max_nan(top, a.m), c);
    float2 s = make_float2(a.s, 0.f), t = make_float2(a.t, 0.f);
#pragma unroll
    for (int k = 0; k < N; k++) add_pair(s, t, x[k], a.m, c);
    a.s = s.x + s.y;
    a.t = t.x + t.y;
}
__device__ __forceinline__ void take_one(Acc &a, float x, float c) {
    const float2 v[1] = {make_float2(x, -CUDART_INF_F)};
    take(a, v, x, c);
}

__device__ __forceinline__ Acc join(const Acc &a, const Acc &b, float c) {
    const float m = max_nan(a.m, b.m);
    const float da = fmaxf((a.m - m) * c, -1e4f), db = fmaxf((b.m - m) * c, -1e4f), fa = ex2(da), fb = ex2(db);
    return Acc{m, a.s * fa + b.s * fb, fa * fmaf(da, a.s, a.t) + fb * fmaf(db, b.s, b.t)};
}
template <int G> __device__ __forceinline__ Acc group_join(Acc a, float c) {
#pragma unroll
    for (int o = G / 2; o; o >>= 1) {
        const Acc b{__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o),
                    __shfl_xor_sync(0xffffffffu, a.t, o)};
        a = threadIdx.x & o ? join(b, a, c) : join(a, b, c);  // the same operands in the same order on both sides
    }
    return a;
}

struct Out {
    const int64_t *tokens;
    int top;
    float *logp, *entropy, *stats;
    int64_t *top_tokens;
    float *top_logp;
};

// What one thread writes for a row: `token` and its masked logit tv.
__device__ __forceinline__ float write_row(const Out &o, int64_t r, int vocab, const Acc &a, int64_t token, float tv,
                                           float inv_t) {
    const bool empty = a.m == -CUDART_INF_F;
    const float log_sum = empty ? -CUDART_INF_F : a.m < CUDART_INF_F ? logf(a.s) : CUDART_NAN_F;
    if (o.entropy) o.entropy[r] = empty ? 0.f : a.m < CUDART_INF_F ? log_sum - a.t / a.s * LN2 : CUDART_NAN_F;
    if (o.stats) {
        o.stats[2 * r] = a.m;
        o.stats[2 * r + 1] = log_sum;
    }
    if (o.logp)
        o.logp[r] = token < 0               ? 0.f
                    : token >= vocab        ? CUDART_NAN_F
                    : tv == -CUDART_INF_F   ? -CUDART_INF_F
                                            : (tv - a.m) * inv_t - log_sum;
    return log_sum;
}
__device__ __forceinline__ void write_top(const Out &o, int64_t r, int q, uint64_t c, float m, float log_sum,
                                          float inv_t) {
    const bool none = key_of(c) == 0u;
    o.top_tokens[r * o.top + q] = none ? -1 : index_of(c);
    o.top_logp[r * o.top + q] = none ? -CUDART_INF_F : (logit_of(c) - m) * inv_t - log_sum;
}

template <class T>
__device__ __forceinline__ float logit_at(const T *x, const uint8_t *legal, int j) {
    return !legal || (legal[j >> 3] >> (j & 7) & 1) ? to_f32(x[j]) : -CUDART_INF_F;
}

// ---------------------------------------------------------------- 16-byte vectors of a row

template <class T> struct Wide;
template <> struct Wide<float> {
    static constexpr int N = 4, LOW_BIT = 0;
    static __device__ __forceinline__ void unpack(const uint4 &v, float2 *x) {
        x[0] = make_float2(__uint_as_float(v.x), __uint_as_float(v.y));
        x[1] = make_float2(__uint_as_float(v.z), __uint_as_float(v.w));
    }
    static __device__ __forceinline__ uint4 pack(const float2 *x) {
        return make_uint4(__float_as_uint(x[0].x), __float_as_uint(x[0].y), __float_as_uint(x[1].x), __float_as_uint(x[1].y));
    }
    static __device__ __forceinline__ uint4 mask(uint4 v, uint32_t bits) {
        const uint32_t none = 0xff800000u;
        return make_uint4(bits & 1 ? v.x : none, bits & 2 ? v.y : none, bits & 4 ? v.z : none, bits & 8 ? v.w : none);
    }
    template <int U> static __device__ __forceinline__ float top(const uint4 (&v)[U]) {
        float m = -CUDART_INF_F;
#pragma unroll
        for (int u = 0; u < U; u++)
            m = max_nan(m, max_nan(max_nan(__uint_as_float(v[u].x), __uint_as_float(v[u].y)), max_nan(__uint_as_float(v[u].z), __uint_as_float(v[u].w))));
        return m;
    }
};
// Two 16-bit types: NONE is -inf.
template <class H2, uint32_t NONE> struct Wide16 {
    static constexpr int N = 8;
    // The 8 bits spread to the top bits of 8 bytes, then a byte's top bit over a half.
    template <int SELECT> static __device__ __forceinline__ uint32_t signs(uint32_t v) {
        uint32_t w;
        asm("prmt.b32 %0, %1, 0, %2;" : "=r"(w) : "r"(v), "n"(SELECT));
        return w;
    }
    static __device__ __forceinline__ uint4 mask(uint4 v, uint32_t bits) {
        const uint32_t lo = (bits & 15u) * 0x10204080u, hi = (bits >> 4 & 15u) * 0x10204080u, none = NONE | NONE << 16;
        const uint32_t a = signs<0x9988>(lo), b = signs<0xbbaa>(lo), c = signs<0x9988>(hi), d = signs<0xbbaa>(hi);
        return make_uint4((v.x & a) | (none & ~a), (v.y & b) | (none & ~b), (v.z & c) | (none & ~c), (v.w & d) | (none & ~d));
    }
    static __device__ __forceinline__ H2 as(const uint32_t &v) { return *reinterpret_cast<const H2 *>(&v); }
    template <int U> static __device__ __forceinline__ float top(const uint4 (&v)[U]) {
        H2 m = __hmax2_nan(__hmax2_nan(as(v[0].x), as(v[0].y)), __hmax2_nan(as(v[0].z), as(v[0].w)));
#pragma unroll
        for (int u = 1; u < U; u++)
            m = __hmax2_nan(m, __hmax2_nan(__hmax2_nan(as(v[u].x), as(v[u].y)), __hmax2_nan(as(v[u].z), as(v[u].w))));
        return max_nan(to_f32(low_of(m)), to_f32(high_of(m)));
    }
    static __device__ __forceinline__ __nv_bfloat16 low_of(__nv_bfloat162 h) { return h.x; }
    static __device__ __forceinline__ __nv_bfloat16 high_of(__nv_bfloat162 h) { return h.y; }
    static __device__ __forceinline__ __half low_of(__half2 h) { return __low2half(h); }
    static __device__ __forceinline__ __half high_of(__half2 h) { return __high2half(h); }
};
template <> struct Wide<__nv_bfloat16> : Wide16<__nv_bfloat162, 0xff80u> {
    static constexpr int LOW_BIT = 16;
    static __device__ __forceinline__ void unpack(const uint4 &v, float2 *x) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 4; k++) x[k] = make_float2(__uint_as_float(w[k] << 16), __uint_as_float(w[k] & 0xffff0000u));
    }
    static __device__ __forceinline__ uint4 pack(const float2 *x) {
        uint4 v;
        __nv_bfloat162 *h = reinterpret_cast<__nv_bfloat162 *>(&v);
#pragma unroll
        for (int k = 0; k < 4; k++) h[k] = __float22bfloat162_rn(x[k]);
        return v;
    }
};
template <> struct Wide<__half> : Wide16<__half2, 0xfc00u> {
    static constexpr int LOW_BIT = 13;
    static __device__ __forceinline__ void unpack(const uint4 &v, float2 *x) {
        const __half2 *h = reinterpret_cast<const __half2 *>(&v);
#pragma unroll
        for (int k = 0; k < 4; k++) x[k] = __half22float2(h[k]);
    }
    static __device__ __forceinline__ uint4 pack(const float2 *x) {
        uint4 v;
        __half2 *h = reinterpret_cast<__half2 *>(&v);
#pragma unroll
        for (int k = 0; k < 4; k++) h[k] = __float22half2_rn(x[k]);
        return v;
    }
};

// A row as 16-byte vectors from its first aligned element `head` on, and the
// elements before and after them (fewer than 2 N).
template <class T> struct Row {
    static constexpr int N = Wide<T>::N;
    const T *x;
    const uint8_t *legal;
    int vocab, head, vectors, loose;
    __device__ __forceinline__ Row(const T *x_, const uint8_t *legal_, int vocab_) : x(x_), legal(legal_), vocab(vocab_) {
        const int to_aligned = (int)((16u - ((uint32_t)reinterpret_cast<uintptr_t>(x) & 15u)) & 15u) / (int)sizeof(T);
        head = to_aligned < vocab ? to_aligned : vocab;
        vectors = (vocab - head) / N;
        loose = vocab - vectors * N;
    }
    __device__ __forceinline__ int first(int i) const { return head + i * N; }
    __device__ __forceinline__ int loose_index(int k) const { return k < head ? k : k + vectors * N; }
    __device__ __forceinline__ uint4 load(int i) const { return __ldg(reinterpret_cast<const uint4 *>(x + first(i))); }
    // the same where the kernel may write over the row
    __device__ __forceinline__ uint4 load_own(int i) const { return *reinterpret_cast<const uint4 *>(x + first(i)); }
    // The legal bits of vector i: its N bits lie in one byte (in all of a row's
    // vectors, where the first starts at a multiple of N) or in two.
    __device__ __forceinline__ uint32_t bits(int i) const {
        const int j = first(i), at = j >> 3;
        uint32_t b = __ldg(legal + at);
        if (head % N) b |= __ldg(legal + ((j + N - 1) >> 3)) << 8;  // the same byte again where one holds them all
        return b >> (j & 7);
    }
};

template <class T, int U> __device__ __forceinline__ float take_vectors(Acc &a, const uint4 (&v)[U], float c, int count = U) {
    constexpr int N = Wide<T>::N;
    const float top = Wide<T>::top(v);
    rescale(a, max_nan(top, a.m), c);
    float2 s = make_float2(a.s, 0.f), t = make_float2(a.t, 0.f);
#pragma unroll
    for (int u = 0; u < U; u++) {
        if (u >= count) break;
        float2 x[N / 2];
        Wide<T>::unpack(v[u], x);
#pragma unroll
        for (int k = 0; k < N / 2; k++) add_pair(s, t, x[k], a.m, c);
    }
    a.s = s.x + s.y;
    a.t = t.x + t.y;
    return top;
}
// The largest logit of each `group` batches of a thread's vectors, a place every
// THREADS floats (or nowhere).
struct Cells {
    float *cell;
    int group, batch;
    float largest;
    __device__ __forceinline__ Cells(float *c, int g) : cell(c), group(g), batch(0) { largest = -CUDART_INF_F; }
    __device__ __forceinline__ void seen(float top, bool end) {
        if (!cell) return;
        largest = max_nan(largest, top);
        if (end && ++batch == group) {
            *cell = largest;
            cell += THREADS;
            largest = -CUDART_INF_F;
            batch = 0;
        }
    }
    __device__ __forceinline__ void finish() {
        if (cell) *cell = largest;
    }
};
// The thread's vectors first, first + STEP, ... below `hi`.
template <class T, bool MASK, int STEP> __device__ __forceinline__ void take_range(Acc &a, const Row<T> &row, int first, int hi, float c, Cells &cells) {
    constexpr int U = UNROLL;
    int i = first;
    // whole batches of the warp's last lane
    for (const int last = 31 - (int)(threadIdx.x & 31); i + last + (U - 1) * STEP < hi; i += U * STEP) {
        uint4 v[U];
#pragma unroll
        for (int u = 0; u < U; u++) v[u] = row.load(i + u * STEP);
        if (MASK) {
            uint32_t b[U];
#pragma unroll
            for (int u = 0; u < U; u++) b[u] = row.bits(i + u * STEP);
#pragma unroll
            for (int u = 0; u < U; u++) v[u] = Wide<T>::mask(v[u], b[u]);
        }
        cells.seen(take_vectors<T>(a, v, c), true);
    }
    if (const int w = i - (int)(threadIdx.x & 31); w < hi) {  // what is left for any lane of the warp: a batch with gaps
        uint4 v[U];
        uint32_t b[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            v[u] = make_uint4(0u, 0u, 0u, 0u);
            b[u] = 0u;
            if (i + u * STEP < hi) {
                v[u] = row.load(i + u * STEP);
                b[u] = MASK ? row.bits(i + u * STEP) : ~0u;
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) v[u] = Wide<T>::mask(v[u], b[u]);
        cells.seen(take_vectors<T>(a, v, c, (hi - w + STEP - 1) / STEP), false);
    }
}
template <class T, bool MASK, int STEP> __device__ __forceinline__ void take_range(Acc &a, const Row<T> &row, int first, int hi, float c) {
    Cells none(nullptr, 1);
    take_range<T, MASK, STEP>(a, row, first, hi, c, none);
}

// ---------------------------------------------------------------- one warp's share of the work on a row

constexpr int WARP_CAP = 512;
struct WarpShared {
    uint64_t list[WARP_CAP], best[MAX_TOP];
    uint16_t column[THREADS];
    int count, cells;
};
constexpr int CELLS = 12, CELL_CAP = 512;  // cells of a thread's vectors in a long row; cells that a warp looks at
struct CellShared {
    uint16_t cell[CELL_CAP];
};

// The join of EACH accumulators of each lane: the largest maximum first, then
// the sums at its scale. Every lane gets it.
template <int EACH> __device__ __forceinline__ Acc warp_join(const Acc (&a)[EACH], float c) {
    float m = a[0].m;
#pragma unroll
    for (int i = 1; i < EACH; i++) m = max_nan(m, a[i].m);
#pragma unroll
    for (int o = 16; o; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    float s = 0.f, t = 0.f;
#pragma unroll
    for (int i = 0; i < EACH; i++) {
        const float d = fmaxf((a[i].m - m) * c, -1e4f), f = ex2(d);
        s = fmaf(a[i].s, f, s);
        t = fmaf(f, fmaf(d, a[i].s, a[i].t), t);
    }
    return Acc{m, warp_sum(s), warp_sum(t)};
}

// A bound found down to bit LOW_BIT, as a key: the bits below are those of every key of
// its sign (16-bit numbers fill only the upper ones, and a negative one's key is its
// complement), so that equal logits compare equal to it; at least 1.
template <int LOW_BIT> __device__ __forceinline__ uint32_t whole_bound(uint32_t bound) {
    return bound == 0u ? 1u : bound & 0x80000000u ? bound : bound | ((1u << LOW_BIT) - 1u);
}
// A bound that at least `top` of the warp's keys reach, and seldom many more (or
// 1, which every token reaches): bisection, by ballots where a lane has one key,
// else two bits at a time with three counts (below 1,024) in one sum.
template <int EACH, int LOW_BIT> __device__ __forceinline__ uint32_t bound_of(const uint32_t (&key)[EACH], int top) {
    uint32_t bound = 0u;
    if constexpr (EACH == 1) {
        for (int bit = 31; bit >= LOW_BIT; bit--) {
            const uint32_t next = bound | 1u << bit;
            const int n = __popc(__ballot_sync(0xffffffffu, key[0] >= next));
            if (n < top) continue;
            bound = next;
            if (n <= top + top / 4) break;
        }
    } else {
        auto reach = [&](uint32_t b) {
            int n = 0;
#pragma unroll
            for (int i = 0; i < EACH; i++) n += key[i] >= b;
            return n;
        };
        for (int bit = 30; bit >= (LOW_BIT & ~1); bit -= 2) {
            const uint32_t b1 = bound | 1u << bit, b2 = bound | 2u << bit, b3 = bound | 3u << bit;
            const int n = __reduce_add_sync(0xffffffffu, reach(b1) | reach(b2) << 10 | reach(b3) << 20);
            const int n1 = n & 1023, n2 = n >> 10 & 1023, n3 = n >> 20;
            if (n1 < top) continue;
            bound = n3 >= top ? b3 : n2 >= top ? b2 : b1;
            if ((n3 >= top ? n3 : n2 >= top ? n2 : n1) <= top + top / 4) break;
        }
    }
    return whole_bound<LOW_BIT>(bound);
}

// The row's best `top` candidates, into w.best, by one warp. seen[i]: the largest
// logit among vectors lane + 32 i, lane + 32 i + 32 EACH, ... of the row; cell
// (long rows): the same for each `group` batches of them.
template <class T, bool MASK, int EACH>
__device__ __forceinline__ void warp_select(WarpShared &w, const Row<T> &row, const float (&seen)[EACH], int top, const float *cell, int group,
                                            CellShared *cs) {
    constexpr int N = Wide<T>::N, STEP = 32 * EACH;
    const int lane = threadIdx.x & 31;
    uint32_t key[EACH];
#pragma unroll
    for (int i = 0; i < EACH; i++) key[i] = order_key(seen[i]);
    const uint32_t bound = bound_of<EACH, Wide<T>::LOW_BIT>(key, top);
    // as a logit: not below it is what reaches the bound (and a NaN)
    const float least = bound < 0x00800000u ? -3.402823466e38f : logit_of((uint64_t)bound << 32);
    int columns = 0;
#pragma unroll
    for (int i = 0; i < EACH; i++) {
        const uint32_t in = __ballot_sync(0xffffffffu, key[i] >= bound);
        if (key[i] >= bound) w.column[columns + __popc(in & ((1u << lane) - 1u))] = (uint16_t)(lane + 32 * i);
        columns += __popc(in);
    }
    if (lane == 0) w.count = 0;
    w.best[lane] = 0u;
    __syncwarp();
    auto put = [&](uint32_t k, int j) {
        const int at = atomicAdd(&w.count, 1);
        if (at < WARP_CAP) w.list[at] = candidate(k, j);
    };
    auto vector = [&](int i, float2 (&x)[N / 2]) {
        uint4 v = row.load(i);
        if (MASK) v = Wide<T>::mask(v, row.bits(i));
        Wide<T>::unpack(v, x);
    };
    auto element = [&](const float2 (&x)[N / 2], int k) { return order_key(k & 1 ? x[k / 2].y : x[k / 2].x); };
    auto loose = [&](int k) { return order_key(logit_at(row.x, MASK ? row.legal : nullptr, row.loose_index(k))); };
    auto look = [&](int i, uint4 v) {
        if (MASK) v = Wide<T>::mask(v, row.bits(i));
        const uint4 one[1] = {v};
        if (Wide<T>::top(one) < least) return;
        float2 x[N / 2];
        Wide<T>::unpack(v, x);
#pragma unroll
        for (int k = 0; k < N; k++)
            if (!((k & 1 ? x[k / 2].y : x[k / 2].x) < least)) {
                const uint32_t e = element(x, k);
                if (e >= bound) put(e, row.first(i) + k);
            }
    };
    bool many = false;
    int deep = (row.vectors + STEP - 1) / STEP, cells = columns;
    if (EACH > 1) {  // of the columns' cells, those that reach the bound
        if (lane == 0) w.cells = 0;
        __syncwarp();
        const int span = UNROLL * group, parts = (deep + span - 1) / span;
        for (int i = lane / 8; i < columns; i += 4)
            for (int p = lane % 8; p < parts; p += 8) {
                const int col = w.column[i];
                if (cell[p * THREADS + col] < least) continue;
                const int at = atomicAdd(&w.cells, 1);
                if (at < CELL_CAP) cs->cell[at] = (uint16_t)(p << 8 | col);
            }
        __syncwarp();
        cells = w.cells;
        many = cells > CELL_CAP;
        deep = span;
    }
    if (!many)
        for (int it0 = 0; it0 < cells * deep; it0 += 64) {
            uint4 v[2];
            int i[2];
#pragma unroll
            for (int u = 0; u < 2; u++) {
                i[u] = row.vectors;
                if (it0 + 32 * u >= cells * deep) continue;
                const int it = it0 + 32 * u + lane, k = it / deep, q = it - k * deep;
                if (it < cells * deep) {
                    if (EACH > 1) {
                        const int id = cs->cell[k];
                        i[u] = (id & 255) + ((id >> 8) * deep + q) * STEP;
                    } else
                        i[u] = w.column[k] + q * STEP;
                }
                if (i[u] < row.vectors) v[u] = row.load(i[u]);
            }
#pragma unroll
            for (int u = 0; u < 2; u++)
                if (i[u] < row.vectors) look(i[u], v[u]);
        }
    if (lane < row.loose) {
        const uint32_t e = loose(lane);
        if (e >= bound) put(e, row.loose_index(lane));
    }
    __syncwarp();
    if (many || w.count > WARP_CAP) {
        // Many equal logits: the row once more from its start, with what is above the bound and the first that equal it.
        __syncwarp();
        if (lane == 0) w.count = 0;
        __syncwarp();
        int equal = 0;  // of those, how many are in the list
        auto more = [&](uint32_t e, int j) {
            const bool in = e > bound || (e == bound && equal < top);
            if (in) put(e, j);
        };
        const int tail = row.loose - row.head;
        {
            const uint32_t e = lane < row.head ? loose(lane) : 0u;
            more(e, lane);
            equal += __popc(__ballot_sync(0xffffffffu, e == bound));
        }
        for (int i0 = 0; i0 < row.vectors; i0 += 32) {
            const int i = i0 + lane;
            int here = 0;
            if (i < row.vectors) {
                float2 x[N / 2];
                vector(i, x);
#pragma unroll
                for (int k = 0; k < N; k++) {
                    const uint32_t e = element(x, k);
                    more(e, row.first(i) + k);
                    here += e == bound;
                }
            }
            equal += __reduce_add_sync(0xffffffffu, here);
        }
        const uint32_t e = lane < tail ? loose(row.head + lane) : 0u;
        more(e, row.loose_index(row.head + lane));
        __syncwarp();
    }
    const int n = w.count;
    if (n <= WARP_CAP) {
        for (int i = lane; i < n; i += 32) {  // a candidate's place is the number of better ones
            const uint64_t d = w.list[i];
            int place = 0;
            for (int q = 0; q < n; q++) place += w.list[q] > d;
            if (place < top) w.best[place] = d;
        }
    } else {  // hundreds above the bound: round by round
        uint64_t last = ~0ull;
        for (int q = 0; q < top; q++) {
            uint64_t b = 0u;
            auto consider = [&](uint32_t e, int j) {
                const uint64_t d = candidate(e, j);
                if (d < last && d > b) b = d;
            };
            for (int i = lane; i < row.vectors; i += 32) {
                float2 x[N / 2];
                vector(i, x);
#pragma unroll
                for (int k = 0; k < N; k++) consider(element(x, k), row.first(i) + k);
            }
            if (lane < row.loose) consider(loose(lane), row.loose_index(lane));
#pragma unroll
            for (int o = 16; o; o >>= 1) b = max(b, (uint64_t)__shfl_xor_sync(0xffffffffu, b, o));
            if (lane == 0) w.best[q] = b;
            last = b;
        }
    }
    __syncwarp();
}

// All of a row's outputs, by one warp. tv: the token's masked logit.
template <class T, bool MASK, int EACH>
__device__ __forceinline__ void warp_finish(WarpShared &w, const Row<T> &row, const Acc (&own)[EACH], const float (&seen)[EACH], const Out &out,
                                            int64_t r, int64_t token, float tv, float inv_t, const float *cell = nullptr, int group = 1,
                                            CellShared *cs = nullptr) {
    const Acc a = warp_join(own, inv_t * LOG2E);
    const int lane = threadIdx.x & 31;
    const float log_sum = a.m == -CUDART_INF_F ? -CUDART_INF_F : a.m < CUDART_INF_F ? logf(a.s) : CUDART_NAN_F;
    if (lane == 0) write_row(out, r, row.vocab, a, token, tv, inv_t);
    if (out.top) {
        warp_select<T, MASK, EACH>(w, row, seen, out.top, cell, group, cs);
        if (lane < out.top) write_top(out, r, lane, w.best[lane], a.m, log_sum, inv_t);
        __syncwarp();
    }
}
template <class T> __device__ __forceinline__ void token_of(const Out &out, const Row<T> &row, int64_t r, int64_t &token, float &tv) {
    token = out.logp ? out.tokens[r] : -1;
    tv = token >= 0 && token < row.vocab ? logit_at(row.x, row.legal, (int)token) : -CUDART_INF_F;
}

// Middling rows: a warp each, so that nothing waits for a barrier. With few vectors
// a lane, the joins and the alternatives are what it costs: 16,384 rows of 4,099
// in fp16 with 5 of them take 45 us (46 % of a copy's rate), 65,536 of 1,000 in
// bf16 81 us (26 %; 91 with 8, 78 % of the issue slots). (A block a row: 218 and 517 us.)
template <class T, bool MASK>
__global__ void __launch_bounds__(THREADS, 5)
    warp_forward_kernel(const T *__restrict__ logits, int64_t ld, int64_t rows, int vocab,
                        const uint8_t *__restrict__ legal, int64_t ldlegal, float inv_t, Out out) {
    __shared__ WarpShared shared[WARPS];
    WarpShared &w = shared[threadIdx.x >> 5];
    const int lane = threadIdx.x & 31;
    const float c = inv_t * LOG2E;
    for (int64_t r = (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5); r < rows; r += (int64_t)gridDim.x * WARPS) {
        const Row<T> row(logits + r * ld, MASK ? legal + r * ldlegal : nullptr, vocab);
        int64_t token;
        float tv;
        token_of(out, row, r, token, tv);
        Acc a[1] = {{-CUDART_INF_F, 0.f, 0.f}};
        take_range<T, MASK, 32>(a[0], row, lane, row.vectors, c);
        const float seen[1] = {a[0].m};
        if (lane < row.loose) take_one(a[0], logit_at(row.x, row.legal, row.loose_index(lane)), c);
        warp_finish<T, MASK, 1>(w, row, a, seen, out, r, token, tv, inv_t);
    }
}

// Long rows: eight warps of a block read row after row and leave each thread's
// sums in shared memory, where two more join them and find the alternatives while
// the eight read on. Each of the two has a place for one row's sums, and a pair
// of barriers that hand it over and back. (Without them the blocks' reading
// stopped for each row's alternatives: 4,096 rows of 32,768 in bf16 took 87 us.)
// They take 66 us with 8 alternatives (4.0 TB/s, 62 % of a copy's rate), 56 without,
// 78 with a mask and 91 with both. Its bounds lie close together: the exponentials alone take
// 30 us at 16 a clock and SM, half of the issue slots are used, and more bytes on
// their way (copies into shared memory two batches ahead) cost the L1 that the
// alternatives and masks are read through: 69 to 100 us.
struct LongShared {
    float m[2][THREADS], s[2][THREADS], t[2][THREADS], seen[2][THREADS], cell[2][CELLS + 1][THREADS];
    WarpShared warp[2];
    CellShared cells[2];
};
__device__ __forceinline__ void bar_sync(int id) { asm volatile("barrier.sync %0, %1;" ::"r"(id), "n"(THREADS + 32) : "memory"); }
__device__ __forceinline__ void bar_arrive(int id) { asm volatile("barrier.arrive %0, %1;" ::"r"(id), "n"(THREADS + 32) : "memory"); }

template <class T, bool MASK>
__global__ void __launch_bounds__(THREADS + 64, 4)
    long_forward_kernel(const T *__restrict__ logits, int64_t ld, int64_t rows, int vocab,
                        const uint8_t *__restrict__ legal, int64_t ldlegal, float inv_t, Out out) {
    extern __shared__ __align__(16) unsigned char space[];
    LongShared &sh = *reinterpret_cast<LongShared *>(space);
    const int tid = threadIdx.x, lane = tid & 31;
    const float c = inv_t * LOG2E;
    // batches to a cell, so that a thread has at most CELLS whole ones
    const int group = vocab / (Wide<T>::N * THREADS * UNROLL * CELLS) + 1;
    int turn = 0;
    if (tid < THREADS) {
        for (int64_t r = blockIdx.x; r < rows; r += gridDim.x, turn ^= 1) {
            const Row<T> row(logits + r * ld, MASK ? legal + r * ldlegal : nullptr, vocab);
            Acc a{-CUDART_INF_F, 0.f, 0.f};
            if (r >= blockIdx.x + 2 * (int64_t)gridDim.x) bar_sync(3 + turn);  // the row before the last is done with
            Cells cells(out.top ? &sh.cell[turn][0][tid] : nullptr, group);
            take_range<T, MASK, THREADS>(a, row, tid, row.vectors, c, cells);
            cells.finish();
            const float seen = a.m;
            if (tid < row.loose) take_one(a, logit_at(row.x, row.legal, row.loose_index(tid)), c);
            sh.m[turn][tid] = a.m;
            sh.s[turn][tid] = a.s;
            sh.t[turn][tid] = a.t;
            sh.seen[turn][tid] = seen;
            __threadfence_block();
            bar_arrive(1 + turn);
        }
    } else {
        turn = (tid - THREADS) >> 5;
        for (int64_t r = blockIdx.x + (int64_t)turn * gridDim.x; r < rows; r += 2 * (int64_t)gridDim.x) {
            const Row<T> row(logits + r * ld, MASK ? legal + r * ldlegal : nullptr, vocab);
            int64_t token;
            float tv;
            token_of(out, row, r, token, tv);
            bar_sync(1 + turn);
            Acc a[WARPS];
            float seen[WARPS];
#pragma unroll
            for (int i = 0; i < WARPS; i++) {
                a[i] = Acc{sh.m[turn][lane + 32 * i], sh.s[turn][lane + 32 * i], sh.t[turn][lane + 32 * i]};
                seen[i] = sh.seen[turn][lane + 32 * i];
            }
            warp_finish<T, MASK, WARPS>(sh.warp[turn], row, a, seen, out, r, token, tv, inv_t, &sh.cell[turn][0][0], group, &sh.cells[turn]);
            __syncwarp();
            if (r + 2 * (int64_t)gridDim.x < rows) bar_arrive(3 + turn);
        }
    }
}

// ---------------------------------------------------------------- few long rows: a cluster of 2 to 8 blocks each

// A row over up to 8 SMs, whose sums and candidates the first block reads from the
// others' shared memory. Latency is its bound: 4 rows of 131,072 in bf16, masked, with
// 20 alternatives, take 11 us, one of 262,144 in fp32 with 32 takes 15 us.

struct Shared {
    Acc warp[WARPS], block;
    uint64_t list[CAP], best[MAX_TOP];
    uint32_t keys[THREADS], bound;
    uint16_t column[THREADS];
    int columns, count;
    uint64_t round[WARPS];
};
static_assert(MAX_CLUSTER * MAX_TOP <= CAP, "the cluster's candidates fit the list");

template <class T> __device__ __forceinline__ T *peer(T *p, uint32_t rank) {
    T *q;
    asm("mapa.u64 %0, %1, %2;" : "=l"(q) : "l"(p), "r"(rank));
    return q;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
}

// best[0..top) of list[0..n): each candidate's place is the number of better ones.
__device__ __forceinline__ void order_list(Shared &sh, int n, int top) {
    for (int q = threadIdx.x; q < top; q += THREADS) sh.best[q] = 0u;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += THREADS) {
        const uint64_t c = sh.list[i];
        int place = 0;
        for (int q = 0; q < n; q++) place += sh.list[q] > c;
        if (place < top && key_of(c)) sh.best[place] = c;
    }
    __syncthreads();
}

// The block's best `top` candidates of vectors [lo, hi) (and of the loose
// elements, if they are its), into sh.best. m: the thread's largest logit.
template <class T, bool MASK>
__device__ __forceinline__ void select_top(Shared &sh, const Row<T> &row, int lo, int hi, bool own_loose, float m, int top) {
    constexpr int N = Wide<T>::N, EACH = THREADS / 32;
    const int tid = threadIdx.x;
    sh.keys[tid] = order_key(m);
    __syncthreads();
    if (tid < 32) {  // one warp looks for the bound: the others would only wait for one another more often
        uint32_t key[EACH];
        int some = 0;
#pragma unroll
        for (int i = 0; i < EACH; i++) some += (key[i] = sh.keys[tid + 32 * i]) >= 1u;
        uint32_t bound = 0u;
        if (__reduce_add_sync(0xffffffffu, some) >= top)
            for (int bit = 31; bit >= Wide<T>::LOW_BIT; bit--) {
                const uint32_t next = bound | 1u << bit;
                int n = 0;
#pragma unroll
                for (int i = 0; i < EACH; i++) n += key[i] >= next;
                n = __reduce_add_sync(0xffffffffu, n);
                if (n >= top) {
                    bound = next;
                    if (n <= top + top / 4) break;
                }
            }
        bound = whole_bound<Wide<T>::LOW_BIT>(bound);
        int columns = 0;
#pragma unroll
        for (int i = 0; i < EACH; i++) {
            const uint32_t in = __ballot_sync(0xffffffffu, key[i] >= bound);
            if (key[i] >= bound) sh.column[columns + __popc(in & ((1u << tid) - 1u))] = (uint16_t)(tid + 32 * i);
            columns += __popc(in);
        }
        if (tid == 0) {
            sh.bound = bound;
            sh.columns = columns;
            sh.count = 0;
        }
    }
    __syncthreads();
    const uint32_t bound = sh.bound;
    auto offer = [&](float x, int j) {
        const uint32_t k = order_key(x);
        if (k >= bound) {
            const int at = atomicAdd(&sh.count, 1);
            if (at < CAP) sh.list[at] = candidate(k, j);
        }
    };
    const int columns = sh.columns, items = columns * ((hi - lo + THREADS - 1) / THREADS);
    for (int it = tid; it < items; it += THREADS) {
        const int i = lo + sh.column[it % columns] + it / columns * THREADS;
        if (i >= hi) continue;
        uint4 v = row.load(i);
        if (MASK) v = Wide<T>::mask(v, row.bits(i));
        float2 x[N / 2];
        Wide<T>::unpack(v, x);
#pragma unroll
        for (int k = 0; k < N; k++) offer(k & 1 ? x[k / 2].y : x[k / 2].x, row.first(i) + k);
    }
    if (own_loose && tid < row.loose) {
        const int j = row.loose_index(tid);
        offer(logit_at(row.x, MASK ? row.legal : nullptr, j), j);
    }
    __syncthreads();
    if (sh.count <= CAP) {
        order_list(sh, sh.count, top);
        return;
    }
    uint64_t last = ~0ull;
    for (int q = 0; q < top; q++) {
        uint64_t c = 0u;
        auto consider = [&](float x, int j) {
            const uint64_t d = candidate(order_key(x), j);
            if (d < last && d > c) c = d;
        };
        for (int i = lo + tid; i < hi; i += THREADS) {
            uint4 v = row.load(i);
            if (MASK) v = Wide<T>::mask(v, row.bits(i));
            float2 x[N / 2];
            Wide<T>::unpack(v, x);
#pragma unroll
            for (int k = 0; k < N; k++) consider(k & 1 ? x[k / 2].y : x[k / 2].x, row.first(i) + k);
        }
        if (own_loose && tid < row.loose) {
            const int j = row.loose_index(tid);
            consider(logit_at(row.x, MASK ? row.legal : nullptr, j), j);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) c = max(c, (uint64_t)__shfl_xor_sync(0xffffffffu, c, o));
        __syncthreads();
        if ((tid & 31) == 0) sh.round[tid >> 5] = c;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WARPS; w++) c = max(c, sh.round[w]);
        if (tid == 0) sh.best[q] = c;
        last = c;
    }
    __syncthreads();
}

template <class T, bool MASK>
__global__ void __launch_bounds__(THREADS, 4)
    cluster_forward_kernel(const T *__restrict__ logits, int64_t ld, int64_t rows, int vocab,
                           const uint8_t *__restrict__ legal, int64_t ldlegal, float inv_t, int cluster, Out out) {
    __shared__ Shared sh;
    const int tid = threadIdx.x, rank = blockIdx.x % cluster;
    const float c = inv_t * LOG2E;
    for (int64_t r = blockIdx.x / cluster; r < rows; r += gridDim.x / cluster) {
        const Row<T> row(logits + r * ld, MASK ? legal + r * ldlegal : nullptr, vocab);
        const int lo = (int)((int64_t)row.vectors * rank / cluster), hi = (int)((int64_t)row.vectors * (rank + 1) / cluster);
        int64_t token = -1;
        float tv = -CUDART_INF_F;
        if (rank == 0 && tid == 0 && out.logp) {
            token = out.tokens[r];
            if (token >= 0 && token < vocab) tv = logit_at(row.x, row.legal, (int)token);
        }
        Acc a{-CUDART_INF_F, 0.f, 0.f};
        take_range<T, MASK, THREADS>(a, row, lo + tid, hi, c);
        const float seen = a.m;  // of the vectors alone
        if (rank == 0 && tid < row.loose) {
            take_one(a, logit_at(row.x, row.legal, row.loose_index(tid)), c);
        }
        a = group_join<32>(a, c);
        if ((tid & 31) == 0) sh.warp[tid >> 5] = a;
        if (out.top) select_top<T, MASK>(sh, row, lo, hi, rank == 0, seen, out.top);
        __syncthreads();
        if (tid < 32) a = group_join<WARPS>(sh.warp[tid % WARPS], c);
        if (tid == 0) sh.block = a;
        cluster_sync();
        if (rank == 0) {
            if (tid < 32)
                for (int p = 1; p < cluster; p++) a = join(a, *peer(&sh.block, p), c);
            if (out.top) {
                for (int q = tid; q < cluster * out.top; q += THREADS) {
                    const int p = q / out.top;
                    sh.list[q] = *peer(&sh.best[q - p * out.top], p);
                }
                __syncthreads();
                order_list(sh, cluster * out.top, out.top);
            }
        }
        if (rank == 0) {
            if (tid < 32) {
                const float log_sum = a.m == -CUDART_INF_F ? -CUDART_INF_F : a.m < CUDART_INF_F ? logf(a.s) : CUDART_NAN_F;
                if (tid == 0) write_row(out, r, vocab, a, token, tv, inv_t);
                if (tid < out.top) write_top(out, r, tid, sh.best[tid], a.m, log_sum, inv_t);
            }
        }
        cluster_sync();  // the other blocks' shared memory has been read
    }
}

// ---------------------------------------------------------------- short rows: eight lanes each, in registers

// One read of the row, joins of three steps. 4,096 rows of 28 in fp32, masked, with 4
// alternatives take 6.3 us, which is latency. 65,536 in bf16 take 10.8 us (8 % of a
// copy's rate), 25.8 with 4 alternatives; of 12 tokens 9.7. There the bound is
// instructions, 129 of a warp for each row: a load, a mask byte and an exponential for
// each of 64 tokens whatever the vocabulary, and the waits for a second read of the
// token's logit (65 % of the issue slots).

template <class T>
__global__ void __launch_bounds__(THREADS)
    short_forward_kernel(const T *__restrict__ logits, int64_t ld, int64_t rows, int vocab,
                         const uint8_t *__restrict__ legal, int64_t ldlegal, float inv_t, Out out) {
    constexpr int G = 8, NV = SHORT_VOCAB / G, GROUPS = THREADS / G;
    __shared__ uint64_t lists[GROUPS][SHORT_VOCAB], bests[GROUPS][MAX_TOP];
    __shared__ int counts[GROUPS];
    const int lane = threadIdx.x % G, group = threadIdx.x / G;
    const float c = inv_t * LOG2E;
    const int64_t step = (int64_t)gridDim.x * GROUPS;
    for (int64_t base = (int64_t)blockIdx.x * GROUPS; base < rows; base += step) {  // all lanes of a warp stay together
        const int64_t r = base + group;
        const bool live = r < rows;
        const T *row = logits + (live ? r : 0) * ld;
        const uint8_t *bits = legal ? legal + (live ? r : 0) * ldlegal : nullptr;
        float x[NV], largest = -CUDART_INF_F;
        float2 pairs[NV / 2];
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int j = lane + G * i;
            x[i] = live && j < vocab ? logit_at(row, bits, j) : -CUDART_INF_F;
            largest = max_nan(largest, x[i]);
            if (i & 1) pairs[i / 2] = make_float2(x[i - 1], x[i]);
        }
        Acc a{-CUDART_INF_F, 0.f, 0.f};
        take(a, pairs, largest, c);
        a = group_join<G>(a, c);
        int64_t token = -1;
        float tv = -CUDART_INF_F;
        if (live && out.logp) {
            token = out.tokens[r];
            if (token >= 0 && token < vocab) tv = logit_at(row, bits, (int)token);
        }
        const float log_sum = a.m == -CUDART_INF_F ? -CUDART_INF_F : a.m < CUDART_INF_F ? logf(a.s) : CUDART_NAN_F;
        if (live && lane == 0) write_row(out, r, vocab, a, token, tv, inv_t);
        if (!out.top) continue;
        if (lane == 0) counts[group] = 0;
        for (int q = lane; q < out.top; q += G) bests[group][q] = 0u;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const uint32_t k = order_key(x[i]);
            if (k) lists[group][atomicAdd(&counts[group], 1)] = candidate(k, lane + G * i);
        }
        __syncwarp();
        const int n = counts[group];
        for (int i = lane; i < n; i += G) {
            const uint64_t d = lists[group][i];
            int place = 0;
            for (int q = 0; q < n; q++) place += lists[group][q] > d;
            if (place < out.top) bests[group][place] = d;
        }
        __syncwarp();
        if (live)
            for (int q = lane; q < out.top; q += G) write_top(out, r, q, bests[group][q], a.m, log_sum, inv_t);
        __syncwarp();
    }
}

// ---------------------------------------------------------------- gradient

struct Grads {
    const int64_t *tokens;
    const float *stats, *entropy, *dlogp, *dentropy;
};

// A row's constants: with z2 = (x - m) c - l2 = log2 p, dlogits = p (w0 + w1 z2), plus `hit` at the token.
struct RowGrad {
    float m, l2, w0, w1, hit;
    int token;
    bool zero;
};
template <class T>
__device__ __forceinline__ RowGrad row_grad(const Grads &g, const T *x, const uint8_t *legal, int64_t r, int vocab, float inv_t) {
    RowGrad k;
    // With a NaN or +inf in the row all is NaN where p is not 0: from the lowest number on, x - m is not
    // negative for any finite x, so that p is 1 or more, while -inf still gives 0.
    const float log_sum = g.stats[2 * r + 1];
    const bool undefined = log_sum != log_sum;
    k.m = undefined ? -3.402823466e38f : g.stats[2 * r];
    k.l2 = undefined ? 0.f : log_sum * LOG2E;
    k.zero = k.m == -CUDART_INF_F;
    const int64_t token = g.dlogp ? g.tokens[r] : -1;
    const float b = g.dentropy ? g.dentropy[r] : 0.f, h = g.dentropy ? g.entropy[r] : 0.f;
    float a = 0.f;
    k.token = -1;
    if (token >= vocab)
        a = CUDART_NAN_F;
    else if (token >= 0 && logit_at(x, legal, (int)token) != -CUDART_INF_F) {
        a = g.dlogp[r];
        k.token = (int)token;
    }
    if (undefined) a = CUDART_NAN_F;
    k.hit = a * inv_t;
    k.w0 = -(a + b * h) * inv_t;
    k.w1 = -b * inv_t * LN2;
    return k;
}
// Of two logits; where p is 0 (a token that is left out, for one) 0 whatever the factor.
__device__ __forceinline__ float2 grad_of(const RowGrad &k, float2 x, float c) {
    const float2 z2 = __ffma2_rn(__fadd2_rn(x, both(-k.m)), both(c), both(-k.l2));
    const float2 p = make_float2(ex2(z2.x), ex2(z2.y)), d = __fmul2_rn(p, __ffma2_rn(z2, both(k.w1), both(k.w0)));
    return make_float2(p.x == 0.f ? 0.f : d.x, p.y == 0.f ? 0.f : d.y);
}
template <class T> __device__ __forceinline__ T grad_one(const RowGrad &k, float x, int j, float c) {
    return from_f32<T>(k.zero ? 0.f : grad_of(k, make_float2(x, x), c).x + (j == k.token ? k.hit : 0.f));
}

// The legal bytes of a long row in shared memory: read there, two byte loads a
// vector cost next to nothing; from global memory they took an eighth of the
// gradient's time (4,096 rows of 50,021 bf16: 166 us, 147 so, 140 with no mask to
// read). The forward pass, whose issue slots are its bound, gains nothing by it.
constexpr int MASK_BYTES = 8192;
struct alignas(16) MaskShared {
    uint8_t bytes[MASK_BYTES + 32];
};
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void wait_copies() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
template <class T> struct StagedMask {
    static constexpr int VECTORS = MASK_BYTES * 8 / Wide<T>::N;  // that one copy can serve
    uint32_t at;  // where byte 0 of the row would be
    // Copies the bytes of vectors [lo, hi) by THREADS threads, whole 16-byte pieces asynchronously.
    __device__ __forceinline__ void fetch(MaskShared &to, const Row<T> &row, int lo, int hi, int t) {
        const int first = row.first(lo) >> 3, last = (row.first(hi) - 1) >> 3;
        const uint8_t *const p = row.legal + first;
        const int from = (int)(reinterpret_cast<uintptr_t>(p) & 15), end = from + last - first + 1, tail = end & ~15;
        const uint32_t base = (uint32_t)__cvta_generic_to_shared(to.bytes);
        at = base + from - first;
        if (lo >= hi) return;
        for (int q = 16 * t; q < end; q += 16 * THREADS)
            if (q >= from && q + 16 <= end)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(base + q), "l"(p - from + q) : "memory");
        if (t < 16 && t >= from && t < end && (from || end < 16)) to.bytes[t] = p[t - from];
        if (t >= 16 && t < 32 && tail && tail + t - 16 < end) to.bytes[tail + t - 16] = p[tail + t - 16 - from];
    }
    __device__ __forceinline__ uint32_t bits(const Row<T> &row, int i) const {
        const int j = row.first(i), k = j >> 3;
        uint32_t b = byte(k);
        if (row.head % Wide<T>::N) b |= byte((j + Wide<T>::N - 1) >> 3) << 8;
        return b >> (j & 7);
    }
    __device__ __forceinline__ uint32_t byte(int k) const {
        uint32_t b;
        asm volatile("ld.shared.u8 %0, [%1];" : "=r"(b) : "r"(at + k) : "memory");
        return b;
    }
};

// The gradient may be written over the logits (IN_PLACE): a thread reads the elements
// that it writes before it writes them, and every thread of a row reads the token's
// logit besides, for the row's constants. So there a row has one team, which waits for
// its slowest reader before it stores; the pointers are not __restrict__, nor are the
// logits read as data that nobody writes. These are kernels of their own, because
// without the promise of __restrict__ the others would lose 1 to 4 %.
template <class T, bool IN_PLACE> struct Apart {
    using In = const T *__restrict__;
    using Result = T *__restrict__;
};
template <class T> struct Apart<T, true> {
    using In = const T *;
    using Result = T *;
};

// A warp or (long rows) a block takes rows or, where they are few, shares of them. The
// vectors are the logits' aligned ones; the gradient is stored as vectors where
// its rows are aligned alike, else element by element. Memory is its bound: 4,096
// rows of 32,768 in bf16 take 88 us (94 % of a copy's rate), 4,096 of 50,021 with
// a mask 146 us (89 %); with rows of a few vectors a lane the constants of each
// row show (65,536 of 1,000: 57 us, 70 %).
template <class T, bool MASK, int TEAM, bool IN_PLACE>
__global__ void __launch_bounds__(THREADS, TEAM == 32 ? 5 : 6)
    long_backward_kernel(typename Apart<T, IN_PLACE>::In logits, int64_t ld, int64_t rows, int vocab,
                         const uint8_t *__restrict__ legal, int64_t ldlegal, float inv_t, Grads g,
                         typename Apart<T, IN_PLACE>::Result dlogits, int64_t ldd) {
    constexpr int N = Wide<T>::N;
    const float c = inv_t * LOG2E;
    constexpr bool STAGED = MASK && TEAM == THREADS;
    __shared__ MaskShared shared[1];
    const int t = threadIdx.x % TEAM;
    for (int64_t r = blockIdx.y * (THREADS / TEAM) + threadIdx.x / TEAM; r < rows; r += gridDim.y * (THREADS / TEAM)) {
        const Row<T> row(logits + r * ld, MASK ? legal + r * ldlegal : nullptr, vocab);
        T *d = dlogits + r * ldd;
        const bool alike = ((reinterpret_cast<uintptr_t>(d) ^ reinterpret_cast<uintptr_t>(row.x)) & 15) == 0;
        const int lo = (int)((int64_t)row.vectors * blockIdx.x / gridDim.x), hi = (int)((int64_t)row.vectors * (blockIdx.x + 1) / gridDim.x);
        const RowGrad k = row_grad(g, row.x, row.legal, r, vocab, inv_t);
        if (IN_PLACE) {
            if (TEAM == THREADS)
                __syncthreads();
            else
                __syncwarp();
        }
        for (int from = lo; from < hi;) {  // at once, or a share of the legal bytes at a time
            const int to = STAGED && from + StagedMask<T>::VECTORS < hi ? from + StagedMask<T>::VECTORS : hi;
            StagedMask<T> mask;
            if (STAGED) {
                __syncthreads();  // the share before this one has been read
                mask.fetch(shared[0], row, from, to, t);
                commit_copies();
                wait_copies<0>();
                __syncthreads();
            }
            for (int i0 = from + t; i0 < to; i0 += UNROLL * TEAM) {
                uint4 v[UNROLL];
                uint32_t bits[UNROLL];
    #pragma unroll
                for (int u = 0; u < UNROLL; u++)
                    if (i0 + u * TEAM < to) {
                        v[u] = IN_PLACE ? row.load_own(i0 + u * TEAM) : row.load(i0 + u * TEAM);
                        if (MASK) bits[u] = STAGED ? mask.bits(row, i0 + u * TEAM) : row.bits(i0 + u * TEAM);
                    }
    #pragma unroll
                for (int u = 0; u < UNROLL; u++) {
                    const int i = i0 + u * TEAM, j = row.first(i);
                    if (i >= to) break;
                    float2 x[N / 2];
                    if (MASK) v[u] = Wide<T>::mask(v[u], bits[u]);
                    Wide<T>::unpack(v[u], x);
    #pragma unroll
                    for (int e = 0; e < N / 2; e++) x[e] = grad_of(k, x[e], c);
                    if ((unsigned)(k.token - j) < (unsigned)N) {
    #pragma unroll
                        for (int e = 0; e < N; e++)
                            if (k.token - j == e) (e & 1 ? x[e / 2].y : x[e / 2].x) += k.hit;
                    }
                    uint4 o = Wide<T>::pack(x);
                    if (k.zero) o = make_uint4(0u, 0u, 0u, 0u);
                    if (alike)
                        *reinterpret_cast<uint4 *>(d + j) = o;
                    else
    #pragma unroll
                        for (int e = 0; e < N; e++) d[j + e] = reinterpret_cast<const T *>(&o)[e];
                }
            }
            from = to;
        }
        if (blockIdx.x == 0 && t < row.loose) {
            const int j = row.loose_index(t);
            d[j] = grad_one<T>(k, logit_at(row.x, row.legal, j), j, c);
        }
    }
}

// Short rows: eight lanes a row. 65,536 of 28, masked, take 10.3 us in fp32 (25 % of a
// copy's rate) and 9.1 in bf16 (16 %), of 12 in bf16 5.8: each lane waits for the row's
// constants, then for one logit and one mask byte at a time (52 % of the issue slots).
template <class T, bool IN_PLACE>
__global__ void __launch_bounds__(THREADS)
    short_backward_kernel(typename Apart<T, IN_PLACE>::In logits, int64_t ld, int64_t rows, int vocab,
                          const uint8_t *__restrict__ legal, int64_t ldlegal, float inv_t, Grads g,
                          typename Apart<T, IN_PLACE>::Result dlogits, int64_t ldd) {
    constexpr int G = 8, GROUPS = THREADS / G;
    const float c = inv_t * LOG2E;
    const int lane = threadIdx.x % G;
    for (int64_t r = (int64_t)blockIdx.x * GROUPS + threadIdx.x / G; r < rows; r += (int64_t)gridDim.x * GROUPS) {
        const T *row = logits + r * ld;
        const uint8_t *bits = legal ? legal + r * ldlegal : nullptr;
        const RowGrad k = row_grad(g, row, bits, r, vocab, inv_t);
        if (IN_PLACE) __syncwarp(0xffu << (threadIdx.x & 24));
        for (int j = lane; j < vocab; j += G) {
            dlogits[r * ldd + j] = grad_one<T>(k, logit_at(row, bits, j), j, c);
        }
    }
}

// ---------------------------------------------------------------- launches

static int blocks_of(int64_t rows, int per_block) {
    const int64_t want = (rows + per_block - 1) / per_block;
    return (int)(want < SMS * 64 ? want : SMS * 64);
}

template <class T>
static int forward(const void *logits, int64_t ld, int64_t rows, int vocab, const uint8_t *legal, int64_t ldlegal,
                   float inv_t, const Out &out, cudaStream_t s) {
    const T *x = (const T *)logits;
    if (vocab <= SHORT_VOCAB) {
        short_forward_kernel<T><<<blocks_of(rows, THREADS / 8), THREADS, 0, s>>>(x, ld, rows, vocab, legal, ldlegal, inv_t, out);
        return (int)cudaGetLastError();
    }
    // a row is split over a cluster while there are too few rows for the 148 SMs (two blocks each) and a
    // block's share stays above two vectors a thread
    int cluster = 1;
    while (cluster < MAX_CLUSTER && rows * cluster < 2 * SMS && vocab / (2 * cluster) >= 2 * THREADS * Wide<T>::N) cluster *= 2;
    if (cluster == 1) {
        if (vocab <= MIDDLE_VOCAB) {
            if (legal)
                warp_forward_kernel<T, true><<<blocks_of(rows, WARPS), THREADS, 0, s>>>(x, ld, rows, vocab, legal, ldlegal, inv_t, out);
            else
                warp_forward_kernel<T, false><<<blocks_of(rows, WARPS), THREADS, 0, s>>>(x, ld, rows, vocab, legal, ldlegal, inv_t, out);
        } else {
            const int grid = (int)(rows < SMS * 4 ? rows : SMS * 4);
            const auto kernel = legal ? long_forward_kernel<T, true> : long_forward_kernel<T, false>;
            if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(LongShared))) return (int)e;
            kernel<<<grid, THREADS + 64, sizeof(LongShared), s>>>(x, ld, rows, vocab, legal, ldlegal, inv_t, out);
        }
        return (int)cudaGetLastError();
    }
    const int64_t most = (1 << 20) / cluster;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = cluster;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((rows < most ? rows : most) * cluster));
    cfg.blockDim = dim3(THREADS);
    cfg.stream = s;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return (int)(legal ? cudaLaunchKernelEx(&cfg, cluster_forward_kernel<T, true>, x, ld, rows, vocab, legal, ldlegal, inv_t, cluster, out)
                       : cudaLaunchKernelEx(&cfg, cluster_forward_kernel<T, false>, x, ld, rows, vocab, legal, ldlegal, inv_t, cluster, out));
}

// A launch of `kernel`, or of `own` where the gradient goes over the logits.
#define D1_LP_BACKWARD(kernel, own, grid)                                                                             \
    do {                                                                                                              \
        if (d == x)                                                                                                   \
            own<<<grid, THREADS, 0, s>>>(x, ld, rows, vocab, legal, ldlegal, inv_t, g, d, ldd);                        \
        else                                                                                                          \
            kernel<<<grid, THREADS, 0, s>>>(x, ld, rows, vocab, legal, ldlegal, inv_t, g, d, ldd);                     \
        return (int)cudaGetLastError();                                                                               \
    } while (0)
template <class T, bool MASK>
static int backward_long(const T *x, int64_t ld, int64_t rows, int vocab, const uint8_t *legal, int64_t ldlegal,
                         float inv_t, const Grads &g, T *d, int64_t ldd, cudaStream_t s) {
    if (vocab / Wide<T>::N <= 32 * UNROLL * 2) {
        const dim3 grid(1, (unsigned)(rows < 65535 * WARPS ? (rows + WARPS - 1) / WARPS : 65535));
        D1_LP_BACKWARD((long_backward_kernel<T, MASK, 32, false>), (long_backward_kernel<T, MASK, 32, true>), grid);
    }
    // blocks for each row: one, or enough of them for the 148 SMs where rows are few
    const int tiles = vocab / (Wide<T>::N * THREADS * UNROLL) + 1;
    const int64_t want = d == x ? 1 : (SMS * 6 + rows - 1) / rows;
    const dim3 grid((unsigned)(want < tiles ? want : tiles), (unsigned)(rows < 65535 ? rows : 65535));
    D1_LP_BACKWARD((long_backward_kernel<T, MASK, THREADS, false>), (long_backward_kernel<T, MASK, THREADS, true>), grid);
}
template <class T>
static int backward(const void *logits, int64_t ld, int64_t rows, int vocab, const uint8_t *legal, int64_t ldlegal,
                    float inv_t, const Grads &g, void *dlogits, int64_t ldd, cudaStream_t s) {
    const T *x = (const T *)logits;
    T *d = (T *)dlogits;
    if (vocab <= SHORT_VOCAB)
        D1_LP_BACKWARD((short_backward_kernel<T, false>), (short_backward_kernel<T, true>), blocks_of(rows, THREADS / 8));
    return legal ? backward_long<T, true>(x, ld, rows, vocab, legal, ldlegal, inv_t, g, d, ldd, s)
                 : backward_long<T, false>(x, ld, rows, vocab, legal, ldlegal, inv_t, g, d, ldd, s);
}

}  // namespace lp
}  // namespace d1

// Of a smaller temperature the reciprocal would not be finite, of an infinite one -inf times it NaN.
static bool temperature_ok(float t) { return t >= FLT_MIN && t <= FLT_MAX; }

extern "C" int d1_token_logprob(const void *logits, int64_t ld, int type, int64_t rows, int vocab,
                                const int64_t *tokens, const void *legal, int64_t ldlegal, float temperature, int top,
                                float *logp, float *entropy, float *stats, int64_t *top_tokens, float *top_logp,
                                void *stream) {
    using namespace d1;
    if (!type_ok(type) || rows < 0 || vocab < 1 || ld < 0 || ldlegal < 0 || !temperature_ok(temperature) || top < 0 ||
        (rows && (!logits || (logp && !tokens) || (top > 0 && (!top_tokens || !top_logp)))) || !element_aligned(logits, type) ||
        !aligned_to(8, tokens, top_tokens) || !aligned_to(4, logp, entropy, stats, top_logp))
        return D1_ERR_BAD_ARGUMENT;
    if (top > lp::MAX_TOP) return D1_ERR_TOO_LARGE;
    if (rows == 0) return 0;
    const float inv_t = 1.f / temperature;
    const lp::Out out{tokens, top, logp, entropy, stats, top_tokens, top_logp};
    const uint8_t *bits = (const uint8_t *)legal;
    const cudaStream_t s = (cudaStream_t)stream;
    if (type == D1_TYPE_F32) return lp::forward<float>(logits, ld, rows, vocab, bits, ldlegal, inv_t, out, s);
    if (type == D1_TYPE_BF16) return lp::forward<__nv_bfloat16>(logits, ld, rows, vocab, bits, ldlegal, inv_t, out, s);
    return lp::forward<__half>(logits, ld, rows, vocab, bits, ldlegal, inv_t, out, s);
}

extern "C" int d1_token_logprob_backward(const void *logits, int64_t ld, int type, int64_t rows, int vocab,
                                         const int64_t *tokens, const void *legal, int64_t ldlegal, float temperature,
                                         const float *stats, const float *entropy, const float *dlogp,
                                         const float *dentropy, void *dlogits, int64_t ldd, void *stream) {
    using namespace d1;
    if (!type_ok(type) || rows < 0 || vocab < 1 || ld < 0 || ldlegal < 0 || !temperature_ok(temperature) ||
        (rows && (!logits || !stats || !dlogits || (dlogp && !tokens) || (dentropy && !entropy))) || ldd < 0 ||
        (rows > 1 && ldd < vocab) || !element_aligned(logits, type) || !element_aligned(dlogits, type) ||
        !aligned_to(8, tokens) || !aligned_to(4, stats, entropy, dlogp, dentropy))
        return D1_ERR_BAD_ARGUMENT;
    if (rows == 0) return 0;
    const int64_t size = type == D1_TYPE_F32 ? 4 : 2;
    if (dlogits == logits ? rows > 1 && ldd != ld
                          : rows_overlap({(uintptr_t)logits, rows, vocab * size, ld * size}, {(uintptr_t)dlogits, rows, vocab * size, ldd * size}))
        return D1_ERR_BAD_ARGUMENT;
    const float inv_t = 1.f / temperature;
    const lp::Grads g{tokens, stats, entropy, dlogp, dentropy};
    const uint8_t *bits = (const uint8_t *)legal;
    const cudaStream_t s = (cudaStream_t)stream;
    if (type == D1_TYPE_F32) return lp::backward<float>(logits, ld, rows, vocab, bits, ldlegal, inv_t, g, dlogits, ldd, s);
    if (type == D1_TYPE_BF16)
        return lp::backward<__nv_bfloat16>(logits, ld, rows, vocab, bits, ldlegal, inv_t, g, dlogits, ldd, s);
    return lp::backward<__half>(logits, ld, rows, vocab, bits, ldlegal, inv_t, g, dlogits, ldd, s);
}
