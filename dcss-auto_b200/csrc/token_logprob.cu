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
// gradient. A NaN or +inf that is not left out makes S, log p and H NaN.
//
// One pass over the logits: each thread keeps a running maximum m, the sum s of
// 2^{(x - m) c} and the sum t of (x - m) c 2^{(x - m) c}, with c = log2(e) / T,
// for a batch of 16-byte vectors at a time (the two sums are scaled down once a
// batch, when the maximum has moved). The joins over threads, warps and the
// blocks of a cluster use the same rule, in a fixed order.
//
// The k alternatives need no second pass over the row. A thread's running
// maximum is the largest of the logits that it saw, so the k-th largest of the
// block's 256 maxima (found by bisection with block-wide counts) bounds the
// k-th largest logit from below, and only threads whose maximum reaches it saw
// a candidate: about k columns of vectors are read again, from L2. The
// candidates (about k of them, unless logits are equal in great numbers) are
// ordered by counting, for each, how many are better. Where more than CAP
// tokens reach the bound, k rounds of a block-wide search replace the list.
#include <math_constants.h>

#include "d1_elem.cuh"

namespace d1 {
namespace lp {

constexpr int THREADS = 256, WARPS = THREADS / 32, MAX_TOP = 32, MAX_CLUSTER = 8, CAP = 768;
constexpr int SMS = 148;
constexpr int UNROLL = 4;           // vectors a thread has in flight
constexpr int SHORT_VOCAB = 1024;   // rows up to here are held in the registers of 8 or 32 lanes
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

// top: the largest of x (a NaN if there is one).
template <int N> __device__ __forceinline__ void take(Acc &a, const float2 (&x)[N], float top, float c) {
    top = max_nan(top, a.m);
    if (!(top <= a.m)) {
        const float d = fmaxf((a.m - top) * c, -1e4f), f = ex2(d);
        a.t = f * fmaf(d, a.s, a.t);
        a.s *= f;
        a.m = top;
    }
    float2 s = make_float2(a.s, 0.f), t = make_float2(a.t, 0.f);
#pragma unroll
    for (int k = 0; k < N; k++) {
        // below 2^-200 the term is zero; the bound also takes in -inf (and -inf - -inf)
        float2 z = __fmul2_rn(__fadd2_rn(x[k], both(-a.m)), both(c));
        z.x = fmaxf(z.x, -200.f);
        z.y = fmaxf(z.y, -200.f);
        const float2 e = make_float2(ex2(z.x), ex2(z.y));
        s = __fadd2_rn(s, e);
        t = __ffma2_rn(z, e, t);
    }
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
    // The legal bits of vector i: its N bits lie in one byte or in two.
    __device__ __forceinline__ uint32_t bits(int i) const {
        const int j = first(i), at = j >> 3, last = (j + N - 1) >> 3;
        const uint32_t lo = __ldg(legal + at), hi = __ldg(legal + last);
        return (lo | hi << 8) >> (j & 7);  // hi is lo itself where one byte holds them all
    }
};

// ---------------------------------------------------------------- long rows: a cluster of 1 to 8 blocks each

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
        bound = max(bound, 1u);
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
    long_forward_kernel(const T *__restrict__ logits, int64_t ld, int64_t rows, int vocab,
                        const uint8_t *__restrict__ legal, int64_t ldlegal, float inv_t, int cluster, Out out) {
    constexpr int N = Wide<T>::N;
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
        int i = lo + tid;
        for (; i + (UNROLL - 1) * THREADS < hi; i += UNROLL * THREADS) {
            uint4 v[UNROLL];
            float2 x[UNROLL * N / 2];
#pragma unroll
            for (int u = 0; u < UNROLL; u++) v[u] = row.load(i + u * THREADS);
#pragma unroll
            for (int u = 0; u < UNROLL; u++) {
                if (MASK) v[u] = Wide<T>::mask(v[u], row.bits(i + u * THREADS));
                Wide<T>::unpack(v[u], x + u * N / 2);
            }
            take(a, x, Wide<T>::top(v), c);
        }
        for (; i < hi; i += THREADS) {
            uint4 v[1] = {row.load(i)};
            float2 x[N / 2];
            if (MASK) v[0] = Wide<T>::mask(v[0], row.bits(i));
            Wide<T>::unpack(v[0], x);
            take(a, x, Wide<T>::top(v), c);
        }
        const float seen = a.m;  // of the vectors alone
        if (rank == 0 && tid < row.loose) {
            take_one(a, logit_at(row.x, row.legal, row.loose_index(tid)), c);
        }
        a = group_join<32>(a, c);
        if ((tid & 31) == 0) sh.warp[tid >> 5] = a;
        if (out.top) select_top<T, MASK>(sh, row, lo, hi, rank == 0, seen, out.top);
        __syncthreads();
        if (tid < 32) a = group_join<WARPS>(sh.warp[tid % WARPS], c);
        if (cluster > 1) {
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
        }
        if (rank == 0) {
            if (tid < 32) {
                const float log_sum = a.m == -CUDART_INF_F ? -CUDART_INF_F : a.m < CUDART_INF_F ? logf(a.s) : CUDART_NAN_F;
                if (tid == 0) write_row(out, r, vocab, a, token, tv, inv_t);
                if (tid < out.top) write_top(out, r, tid, sh.best[tid], a.m, log_sum, inv_t);
            }
        }
        if (cluster > 1)
            cluster_sync();  // the other blocks' shared memory has been read
        else
            __syncthreads();
    }
}

// ---------------------------------------------------------------- short rows: G lanes each, in registers

template <class T, int G, int NV>
__global__ void __launch_bounds__(THREADS)
    short_forward_kernel(const T *__restrict__ logits, int64_t ld, int64_t rows, int vocab,
                         const uint8_t *__restrict__ legal, int64_t ldlegal, float inv_t, Out out) {
    constexpr int GROUPS = THREADS / G, LIST = G * NV < 256 ? G * NV : 256;
    __shared__ uint64_t lists[GROUPS][LIST], bests[GROUPS][MAX_TOP];
    __shared__ int counts[GROUPS];
    const int lane = threadIdx.x % G, group = threadIdx.x / G;
    const uint32_t mates = G == 32 ? 0xffffffffu : ((1u << (G & 31)) - 1u) << (threadIdx.x & 31 & ~(G - 1));
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
        const float seen = a.m;
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
        uint32_t bound = 1u;
        if (G * NV > LIST) {  // else every token fits the list
            const uint32_t key = order_key(seen);
            if (__popc(__ballot_sync(0xffffffffu, key >= 1u) & mates) >= out.top) {
                bound = 0u;
                for (int bit = 31; bit >= Wide<T>::LOW_BIT; bit--) {
                    const uint32_t next = bound | 1u << bit;
                    if (__popc(__ballot_sync(0xffffffffu, key >= next) & mates) >= out.top) bound = next;
                }
                bound = max(bound, 1u);
            }
        }
        if (lane == 0) counts[group] = 0;
        for (int q = lane; q < out.top; q += G) bests[group][q] = 0u;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const uint32_t k = order_key(x[i]);
            if (k >= bound) {
                const int at = atomicAdd(&counts[group], 1);
                if (at < LIST) lists[group][at] = candidate(k, lane + G * i);
            }
        }
        __syncwarp();
        const int n = counts[group];
        if (__any_sync(0xffffffffu, n > LIST)) {  // only where G is a warp: k rounds of a search in registers
            uint64_t last = ~0ull;
            for (int q = 0; q < out.top; q++) {
                uint64_t b = 0u;
#pragma unroll
                for (int i = 0; i < NV; i++) {
                    const uint64_t d = candidate(order_key(x[i]), lane + G * i);
                    if (d < last && d > b) b = d;
                }
#pragma unroll
                for (int o = G / 2; o; o >>= 1) b = max(b, (uint64_t)__shfl_xor_sync(0xffffffffu, b, o));
                if (lane == 0) bests[group][q] = b;
                last = b;
            }
        } else {
            for (int i = lane; i < n; i += G) {
                const uint64_t d = lists[group][i];
                int place = 0;
                for (int q = 0; q < n; q++) place += lists[group][q] > d;
                if (place < out.top) bests[group][place] = d;
            }
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
    k.m = g.stats[2 * r];
    k.l2 = g.stats[2 * r + 1] * LOG2E;
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

// Long rows: a block takes rows (or, where they are few, shares of them). The
// vectors are the logits' aligned ones; the gradient is stored as vectors where
// its rows are aligned alike, else element by element.
template <class T, bool MASK>
__global__ void __launch_bounds__(THREADS, 6)
    long_backward_kernel(const T *__restrict__ logits, int64_t ld, int64_t rows, int vocab,
                         const uint8_t *__restrict__ legal, int64_t ldlegal, float inv_t, Grads g,
                         T *__restrict__ dlogits, int64_t ldd) {
    constexpr int N = Wide<T>::N;
    const float c = inv_t * LOG2E;
    for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
        const Row<T> row(logits + r * ld, MASK ? legal + r * ldlegal : nullptr, vocab);
        T *d = dlogits + r * ldd;
        const bool alike = ((reinterpret_cast<uintptr_t>(d) ^ reinterpret_cast<uintptr_t>(row.x)) & 15) == 0;
        const int lo = (int)((int64_t)row.vectors * blockIdx.x / gridDim.x), hi = (int)((int64_t)row.vectors * (blockIdx.x + 1) / gridDim.x);
        const RowGrad k = row_grad(g, row.x, row.legal, r, vocab, inv_t);
        for (int i0 = lo + threadIdx.x; i0 < hi; i0 += UNROLL * THREADS) {
            uint4 v[UNROLL];
#pragma unroll
            for (int u = 0; u < UNROLL; u++)
                if (i0 + u * THREADS < hi) v[u] = row.load(i0 + u * THREADS);
#pragma unroll
            for (int u = 0; u < UNROLL; u++) {
                const int i = i0 + u * THREADS, j = row.first(i);
                if (i >= hi) break;
                float2 x[N / 2];
                if (MASK) v[u] = Wide<T>::mask(v[u], row.bits(i));
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
        if (blockIdx.x == 0 && threadIdx.x < row.loose) {
            const int j = row.loose_index(threadIdx.x);
            d[j] = grad_one<T>(k, logit_at(row.x, row.legal, j), j, c);
        }
    }
}

// Short rows: G lanes a row.
template <class T, int G>
__global__ void __launch_bounds__(THREADS)
    short_backward_kernel(const T *__restrict__ logits, int64_t ld, int64_t rows, int vocab,
                          const uint8_t *__restrict__ legal, int64_t ldlegal, float inv_t, Grads g,
                          T *__restrict__ dlogits, int64_t ldd) {
    constexpr int GROUPS = THREADS / G;
    const float c = inv_t * LOG2E;
    const int lane = threadIdx.x % G;
    for (int64_t r = (int64_t)blockIdx.x * GROUPS + threadIdx.x / G; r < rows; r += (int64_t)gridDim.x * GROUPS) {
        const T *row = logits + r * ld;
        const uint8_t *bits = legal ? legal + r * ldlegal : nullptr;
        const RowGrad k = row_grad(g, row, bits, r, vocab, inv_t);
#pragma unroll 4
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
        if (vocab <= 64)
            short_forward_kernel<T, 8, 8><<<blocks_of(rows, 32), THREADS, 0, s>>>(x, ld, rows, vocab, legal, ldlegal, inv_t, out);
        else if (vocab <= 256)
            short_forward_kernel<T, 32, 8><<<blocks_of(rows, 8), THREADS, 0, s>>>(x, ld, rows, vocab, legal, ldlegal, inv_t, out);
        else
            short_forward_kernel<T, 32, 32><<<blocks_of(rows, 8), THREADS, 0, s>>>(x, ld, rows, vocab, legal, ldlegal, inv_t, out);
        return (int)cudaGetLastError();
    }
    // a row is split over a cluster while there are too few rows for the 148 SMs (two blocks each) and a
    // block's share stays above two vectors a thread
    int cluster = 1;
    while (cluster < MAX_CLUSTER && rows * cluster < 2 * SMS && vocab / (2 * cluster) >= 2 * THREADS * Wide<T>::N) cluster *= 2;
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
    return (int)(legal ? cudaLaunchKernelEx(&cfg, long_forward_kernel<T, true>, x, ld, rows, vocab, legal, ldlegal, inv_t, cluster, out)
                       : cudaLaunchKernelEx(&cfg, long_forward_kernel<T, false>, x, ld, rows, vocab, legal, ldlegal, inv_t, cluster, out));
}

template <class T>
static int backward(const void *logits, int64_t ld, int64_t rows, int vocab, const uint8_t *legal, int64_t ldlegal,
                    float inv_t, const Grads &g, void *dlogits, int64_t ldd, cudaStream_t s) {
    const T *x = (const T *)logits;
    T *d = (T *)dlogits;
    if (vocab <= SHORT_VOCAB) {
        if (vocab <= 64)
            short_backward_kernel<T, 8><<<blocks_of(rows, 32), THREADS, 0, s>>>(x, ld, rows, vocab, legal, ldlegal, inv_t, g, d, ldd);
        else
            short_backward_kernel<T, 32><<<blocks_of(rows, 8), THREADS, 0, s>>>(x, ld, rows, vocab, legal, ldlegal, inv_t, g, d, ldd);
        return (int)cudaGetLastError();
    }
    // blocks for each row: one, or enough of them for the 148 SMs where rows are few
    const int tiles = vocab / (Wide<T>::N * THREADS * UNROLL) + 1;
    const int64_t want = (SMS * 6 + rows - 1) / rows;
    const dim3 grid((unsigned)(want < tiles ? want : tiles), (unsigned)(rows < 65535 ? rows : 65535));
    if (legal)
        long_backward_kernel<T, true><<<grid, THREADS, 0, s>>>(x, ld, rows, vocab, legal, ldlegal, inv_t, g, d, ldd);
    else
        long_backward_kernel<T, false><<<grid, THREADS, 0, s>>>(x, ld, rows, vocab, legal, ldlegal, inv_t, g, d, ldd);
    return (int)cudaGetLastError();
}

}  // namespace lp
}  // namespace d1

extern "C" int d1_token_logprob(const void *logits, int64_t ld, int type, int64_t rows, int vocab,
                                const int64_t *tokens, const void *legal, int64_t ldlegal, float temperature, int top,
                                float *logp, float *entropy, float *stats, int64_t *top_tokens, float *top_logp,
                                void *stream) {
    using namespace d1;
    if (!type_ok(type) || rows < 0 || vocab < 1 || ld < 0 || ldlegal < 0 || !(temperature > 0.f) || top < 0 ||
        (rows && (!logits || (logp && !tokens) || (top > 0 && (!top_tokens || !top_logp)))) || !element_aligned(logits, type))
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
    if (!type_ok(type) || rows < 0 || vocab < 1 || ld < 0 || ldlegal < 0 || !(temperature > 0.f) ||
        (rows && (!logits || !stats || !dlogits || (dlogp && !tokens) || (dentropy && !entropy))) || ldd < 0 ||
        (rows > 1 && ldd < vocab) || !element_aligned(logits, type) || !element_aligned(dlogits, type))
        return D1_ERR_BAD_ARGUMENT;
    if (rows == 0) return 0;
    const float inv_t = 1.f / temperature;
    const lp::Grads g{tokens, stats, entropy, dlogp, dentropy};
    const uint8_t *bits = (const uint8_t *)legal;
    const cudaStream_t s = (cudaStream_t)stream;
    if (type == D1_TYPE_F32) return lp::backward<float>(logits, ld, rows, vocab, bits, ldlegal, inv_t, g, dlogits, ldd, s);
    if (type == D1_TYPE_BF16)
        return lp::backward<__nv_bfloat16>(logits, ld, rows, vocab, bits, ldlegal, inv_t, g, dlogits, ldd, s);
    return lp::backward<__half>(logits, ld, rows, vocab, bits, ldlegal, inv_t, g, dlogits, ldd, s);
}
