// Log-probabilities of given tokens, with the distribution's entropy and its
// likeliest alternatives, and their gradient (sm_100a).
//
// For one row of logits x over a vocabulary, with z_j = (x_j - max x) / T over
// the legal tokens (legal bit set, or no mask) of finite or infinite logit:
//
//   S = sum_j e^{z_j}     log p_j = z_j - log S     H = log S - sum_j z_j e^{z_j} / S
//   d log p_t / d x_j = (1[j = t] - p_j) / T        d H / d x_j = -p_j (log p_j + H) / T
//
// A token whose bit is clear is left out whatever its logit holds; a logit of
// -inf is left out in the same way. A row with nothing left has log p = -inf,
// H = 0, no alternatives and a zero gradient.
#include <math_constants.h>

#include "d1_elem.cuh"

namespace d1 {
namespace lp {

constexpr int THREADS = 256, WARPS = THREADS / 32, MAX_TOP = 32;

struct Best {
    uint32_t key;  // order_key of the logit; 0: none
    int index;
};

// Whole numbers in the order of the floats, -0 equal to +0 and NaN above all;
// 0 stands for -inf (a token that is left out).
__device__ __forceinline__ uint32_t order_key(float x) {
    if (x != x) return 0xffffffffu;
    if (x == -CUDART_INF_F) return 0u;
    const uint32_t u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ bool better(uint32_t ka, int ia, uint32_t kb, int ib) {
    return ka > kb || (ka == kb && ia < ib);
}

template <class T>
__device__ __forceinline__ float logit_at(const T *x, const uint8_t *legal, int j) {
    return !legal || (legal[j >> 3] >> (j & 7) & 1) ? to_f32(x[j]) : -CUDART_INF_F;
}

__device__ __forceinline__ float block_sum(float x, float *part) {
    x = warp_sum(x);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = x;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < WARPS; i++) s += part[i];
    return s;
}

__device__ __forceinline__ Best block_best(Best b, Best *part) {
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const uint32_t k = __shfl_xor_sync(0xffffffffu, b.key, o);
        const int i = __shfl_xor_sync(0xffffffffu, b.index, o);
        if (better(k, i, b.key, b.index)) b = Best{k, i};
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = b;
    __syncthreads();
    b = part[0];
#pragma unroll
    for (int i = 1; i < WARPS; i++)
        if (better(part[i].key, part[i].index, b.key, b.index)) b = part[i];
    return b;
}

template <class T>
__global__ void __launch_bounds__(THREADS)
    forward_kernel(const T *__restrict__ logits, int64_t ld, int64_t rows, int vocab,
                   const int64_t *__restrict__ tokens, const uint8_t *__restrict__ legal, int64_t ldlegal,
                   float inv_t, int top, float *__restrict__ logp, float *__restrict__ entropy,
                   float *__restrict__ stats, int64_t *__restrict__ top_tokens, float *__restrict__ top_logp) {
    __shared__ float part[WARPS];
    __shared__ Best bests[WARPS];
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const T *x = logits + r * ld;
        const uint8_t *l = legal ? legal + r * ldlegal : nullptr;
        Best b{0u, vocab};
        for (int j = threadIdx.x; j < vocab; j += THREADS) {
            const uint32_t k = order_key(logit_at(x, l, j));
            if (better(k, j, b.key, b.index)) b = Best{k, j};
        }
        b = block_best(b, bests);
        const bool empty = b.key == 0u;
        const float m = empty ? -CUDART_INF_F : to_f32(x[b.index]);
        float s = 0.f, t = 0.f;
        if (!empty)
            for (int j = threadIdx.x; j < vocab; j += THREADS) {
                const float v = logit_at(x, l, j);
                if (v == -CUDART_INF_F) continue;
                const float z = (v - m) * inv_t, e = expf(z);
                s += e;
                t += e > 0.f ? z * e : (z != z ? z : 0.f);
            }
        s = block_sum(s, part);
        t = block_sum(t, part);
        const float log_sum = logf(s);
        if (threadIdx.x == 0) {
            if (entropy) entropy[r] = empty ? 0.f : log_sum - t / s;
            if (stats) {
                stats[2 * r] = m;
                stats[2 * r + 1] = log_sum;
            }
            if (logp) {
                const int64_t tok = tokens[r];
                float v = 0.f;
                if (tok >= vocab)
                    v = CUDART_NAN_F;
                else if (tok >= 0) {
                    v = logit_at(x, l, (int)tok);
                    v = v == -CUDART_INF_F ? v : (v - m) * inv_t - log_sum;
                }
                logp[r] = v;
            }
        }
        for (int q = 0; q < top; q++) {
            if (threadIdx.x == 0) {
                top_tokens[r * top + q] = b.key ? b.index : -1;
                top_logp[r * top + q] = b.key ? (to_f32(x[b.index]) - m) * inv_t - log_sum : -CUDART_INF_F;
            }
            if (q + 1 == top) break;
            Best c{0u, vocab};
            if (b.key)
                for (int j = threadIdx.x; j < vocab; j += THREADS) {
                    const uint32_t k = order_key(logit_at(x, l, j));
                    if (better(b.key, b.index, k, j) && better(k, j, c.key, c.index)) c = Best{k, j};
                }
            b = block_best(c, bests);
        }
    }
}

template <class T>
__global__ void __launch_bounds__(THREADS)
    backward_kernel(const T *__restrict__ logits, int64_t ld, int64_t rows, int vocab,
                    const int64_t *__restrict__ tokens, const uint8_t *__restrict__ legal, int64_t ldlegal,
                    float inv_t, const float *__restrict__ stats, const float *__restrict__ entropy,
                    const float *__restrict__ dlogp, const float *__restrict__ dentropy, T *__restrict__ dlogits,
                    int64_t ldd) {
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const T *x = logits + r * ld;
        const uint8_t *l = legal ? legal + r * ldlegal : nullptr;
        const float m = stats[2 * r], log_sum = stats[2 * r + 1];
        const int64_t tok = tokens ? tokens[r] : -1;
        const bool empty = m == -CUDART_INF_F;
        float a = 0.f, b = dentropy ? dentropy[r] : 0.f, h = dentropy ? entropy[r] : 0.f;
        if (tok >= vocab)
            a = CUDART_NAN_F;
        else if (tok >= 0 && dlogp && logit_at(x, l, (int)tok) != -CUDART_INF_F)
            a = dlogp[r];
        for (int j = threadIdx.x; j < vocab; j += THREADS) {
            const float v = logit_at(x, l, j);
            float d = 0.f;
            if (v != -CUDART_INF_F && !empty) {
                const float lp = (v - m) * inv_t - log_sum, p = expf(lp);
                d = ((j == tok ? a : 0.f) - p * (a + b * ((lp == -CUDART_INF_F ? 0.f : lp) + h))) * inv_t;
            }
            dlogits[r * ldd + j] = from_f32<T>(d);
        }
    }
}

static int grid_of(int64_t rows) { return (int)(rows < 148 * 8 ? rows : 148 * 8); }

}  // namespace lp
}  // namespace d1

extern "C" int d1_token_logprob(const void *logits, int64_t ld, int type, int64_t rows, int vocab,
                                const int64_t *tokens, const void *legal, int64_t ldlegal, float temperature, int top,
                                float *logp, float *entropy, float *stats, int64_t *top_tokens, float *top_logp,
                                void *stream) {
    using namespace d1;
    using namespace d1::lp;
    if (!type_ok(type) || rows < 0 || vocab < 1 || ld < 0 || ldlegal < 0 || !(temperature > 0.f) || top < 0 ||
        (logp && !tokens) || (top > 0 && (!top_tokens || !top_logp)) || (rows && !logits))
        return D1_ERR_BAD_ARGUMENT;
    if (top > MAX_TOP) return D1_ERR_TOO_LARGE;
    if (rows == 0) return 0;
    const float inv_t = 1.f / temperature;
    const cudaStream_t s = (cudaStream_t)stream;
#define D1_LP_FORWARD(T)                                                                                              \
    forward_kernel<T><<<grid_of(rows), THREADS, 0, s>>>((const T *)logits, ld, rows, vocab, tokens,                  \
                                                        (const uint8_t *)legal, ldlegal, inv_t, top, logp, entropy,  \
                                                        stats, top_tokens, top_logp)
    if (type == D1_TYPE_F32)
        D1_LP_FORWARD(float);
    else if (type == D1_TYPE_BF16)
        D1_LP_FORWARD(__nv_bfloat16);
    else
        D1_LP_FORWARD(__half);
    return (int)cudaGetLastError();
}

extern "C" int d1_token_logprob_backward(const void *logits, int64_t ld, int type, int64_t rows, int vocab,
                                         const int64_t *tokens, const void *legal, int64_t ldlegal, float temperature,
                                         const float *stats, const float *entropy, const float *dlogp,
                                         const float *dentropy, void *dlogits, int64_t ldd, void *stream) {
    using namespace d1;
    using namespace d1::lp;
    if (!type_ok(type) || rows < 0 || vocab < 1 || ld < 0 || ldlegal < 0 || !(temperature > 0.f) ||
        (rows && (!logits || !stats || !dlogits)) || (dlogp && !tokens) || (dentropy && !entropy) || ldd < 0 ||
        (rows > 1 && ldd < vocab))
        return D1_ERR_BAD_ARGUMENT;
    if (rows == 0) return 0;
    const float inv_t = 1.f / temperature;
    const cudaStream_t s = (cudaStream_t)stream;
#define D1_LP_BACKWARD(T)                                                                                             \
    backward_kernel<T><<<grid_of(rows), THREADS, 0, s>>>((const T *)logits, ld, rows, vocab, tokens,                 \
                                                         (const uint8_t *)legal, ldlegal, inv_t, stats, entropy,     \
                                                         dlogp, dentropy, (T *)dlogits, ldd)
    if (type == D1_TYPE_F32)
        D1_LP_BACKWARD(float);
    else if (type == D1_TYPE_BF16)
        D1_LP_BACKWARD(__nv_bfloat16);
    else
        D1_LP_BACKWARD(__half);
    return (int)cudaGetLastError();
}
