// Gated linear recurrence over time and its gradient (sm_100a).
//
//   average:  a = sigmoid(g)   h_t = a_t k_t h_{t-1} + (1 - a_t) x_t
//   sum:      a = e^g          h_t = a_t k_t h_{t-1} + x_t
//
// with k_t = 0 where an episode begins at t (reset), else 1; every channel of
// every sequence has its own state. Backward, with E_t = a_t k_t D_t what flows
// from step t to the one before it:
//
//   D_t = dy_t + E_{t+1}    dx_t = (1 - a_t) D_t  or  D_t
//   dg_t = D_t (k_t h_{t-1} - x_t) a_t (1 - a_t)  or  D_t k_t h_{t-1} a_t
//
// States, products of decays and gradients of states are fp32; a 16-bit result
// is rounded once. The gradient reads h_{t-1} as the forward pass stored it
// (rounded to y's type): recomputing it would cost the forward pass again for
// half a rounding step of dg.
//
// Both directions are the map s -> a s + b, whose composition over a chunk of
// steps is again such a map (P, Q); decays of the sum form may pass 1, and their product fp32 where no state does: there P is a
// number and a power of 2. With enough channels one thread walks each
// of them through the whole time, a few steps' loads ahead of the arithmetic.
// With few channels the time is cut into chunks: one launch reduces each chunk
// to its (P, Q), a second runs over the chunks, a third walks all of them side
// by side from their true states. The order of all sums is fixed.
//
// Measured (one B200; floor: each operand once at 6.56 TB/s). 128 steps of 4,096 x 512 channels bf16: 252 us (98 % of the floor's
// rate); 64 steps backward 272 (92 %). 131,072 steps of 256 channels 75 us (floor 31): 34 for the reduction, 35 for the walk, the
// rest the launch between them; 82 in the sum form (70 without the powers). 50,021 x 3 x 111 fp32 backward, sum form, 110 us (51; 105 without).
// One step of 64 x 256: 1.9 us.
//
// A reset replaces the state: a product with 0 would keep an infinity.
#include <initializer_list>
#include <type_traits>

#include "d1_common.cuh"
#include "d1_elem.cuh"
#include "d1_pdl.cuh"

namespace d1 {
namespace gs {

constexpr int SMS = 148, THREADS = 128, CARRY_CHANNELS = 8, CARRY_RUNS = 128, CARRY_EACH = 16;
constexpr int MOST_CHUNKS = CARRY_RUNS * CARRY_EACH;
// P of a chunk with a reset in it: the state before it does not reach its end (decays
// are not negative, and one that has underflowed to 0 still lets an infinity through).
constexpr float CUT = -1.f;
constexpr int MOST_POWER = 1 << 26;  // of P; past this on either side it overflows or removes every state

// A [T, B, D] operand with contiguous channels: strides in elements.
template <class T> struct Span {
    T *p;
    int64_t st, sb;
};

template <class T> struct Args {
    Span<const T> x, gate, y, dy;  // y, dy: backward
    T *out, *dgate;                // y forward; dx backward (contiguous)
    const uint8_t *reset;          // NULL: none
    int64_t reset_t, reset_b;
    const float *start;            // h0 forward, dlast backward (NULL: zeros)
    const float *h0;               // backward: the first step's state (NULL: zeros)
    float *last;                   // last forward, dh0 backward (may be NULL)
    float2 *carry;                 // [chunks][B * D]: (P, Q), then (state before the chunk, -)
    int *power;                    // [chunks][B * D], sum form: the power of 2 that goes with P
    int64_t T_, B, D, lanes;       // lanes = B * D / V
    int64_t size;                  // steps of a chunk
    int chunks;
};

// (a, 1 - a) of the average form from E = e^g, as E / (1 + E) and 1 / (1 + E): neither is a difference from 1. E = 2^x with x = g log2(e)
// rounded, times 1 + (g - x ln 2), which that rounding left out (up to 60 * 2^-24 for large g): right to a few roundings wherever it is a
// normal number. Below, E and a are 0; where 1 / E would vanish E is 2^126, so that 1 - a is 2^-126 at least (a NaN passes).
__device__ __forceinline__ float2 gates(float g) {
    constexpr float LN2 = 0.6931471805599453f, REST = (float)(0.69314718055994530942 - (double)LN2);
    const float x = g * 1.4426950408889634f;
    float e, w, most;
    asm("min.NaN.f32 %0, %1, 0f42FC0000;" : "=f"(most) : "f"(x));  // 126
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(most));
    const float left = fmaf(-x, REST, fmaf(-x, LN2, g));
    if (fabsf(x) < 126.f) e = fmaf(e, left, e);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"(1.f + e));
    return make_float2(e * w, w);
}

// x = x 2^k, 1 <= x < 2, where x is positive and normal; the power is added to `power`.
__device__ __forceinline__ void take_power(float &x, int &power) {
    const uint32_t bits = __float_as_uint(x);
    if (bits - 0x00800000u < 0x7f000000u) {
        power += (int)(bits >> 23) - 127;
        x = __uint_as_float((bits & 0x007fffffu) | 0x3f800000u);
    }
}

// V elements as they lie in memory: words, so that a step under way takes no more registers than its bytes.
template <class T, int V> struct Raw {
    using Word = std::conditional_t<sizeof(T) * V == 2, uint16_t, uint32_t>;
    static constexpr int N = sizeof(T) * V / sizeof(Word);
    struct alignas(sizeof(T) * V) Words {
        Word w[N];
    } r;

    __device__ __forceinline__ void load(const T *p) { r = *reinterpret_cast<const Words *>(p); }
    __device__ __forceinline__ float get(int v) const {
        if constexpr (sizeof(T) == 4)
            return __uint_as_float(r.w[v]);
        else if constexpr (std::is_same_v<T, __nv_bfloat16>)
            return __uint_as_float(V > 1 && v & 1 ? r.w[v / 2] & 0xffff0000u : (uint32_t)r.w[v / 2] << 16);
        else
            return __half2float(__ushort_as_half((unsigned short)(V > 1 && v & 1 ? r.w[v / 2] >> 16 : r.w[v / 2])));
    }
    static __device__ __forceinline__ void store(T *p, const float (&x)[V]) {
        Words o;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int v = 0; v < V; v++) o.w[v] = __float_as_uint(x[v]);
        } else if constexpr (V == 1) {
            const T e = from_f32<T>(x[0]);
            o.w[0] = *reinterpret_cast<const uint16_t *>(&e);
        } else {
#pragma unroll
            for (int v = 0; v < V; v += 2) {
                if constexpr (std::is_same_v<T, __nv_bfloat16>) {
                    const __nv_bfloat162 e = __floats2bfloat162_rn(x[v], x[v + 1]);
                    o.w[v / 2] = *reinterpret_cast<const uint32_t *>(&e);
                } else {
                    const __half2 e = __floats2half2_rn(x[v], x[v + 1]);
                    o.w[v / 2] = *reinterpret_cast<const uint32_t *>(&e);
                }
            }
        }
        *reinterpret_cast<Words *>(p) = o;
    }
};

template <class T, int V> struct Step {  // one step's operands of V channels
    Raw<T, V> x, gate, y, dy;
};

// Where a thread reads and writes: its channels' addresses at its next step, and how far a step moves them.
template <class T, int V, bool SUM, bool BACK, int PART> struct Walk {
    const T *x, *gate, *y, *dy;
    T *out, *dgate;
    int64_t sx, sgate, sy, sdy, sout;

    __device__ __forceinline__ void load(Step<T, V> &s) {
        s.gate.load(gate);
        gate += sgate;
        if constexpr (!BACK || (PART == 1 && !SUM)) {
            s.x.load(x);
            x += sx;
        }
        if constexpr (BACK) {
            s.dy.load(dy);
            dy += sdy;
        }
    }
    __device__ __forceinline__ void load_before(Step<T, V> &s) {  // y of the step before (backward)
        s.y.load(y);
        y += sy;
    }
};

// Blocks of a kernel that an SM holds at once (their registers are limited to that).
constexpr int blocks_of(int V, bool back, int part) { return V == 1 ? (back && part ? 5 : 6) : back && part ? 3 : 5; }

// PART 0: reduce a chunk; 1: walk it. A thread has V channels of one sequence in one chunk of the time.
template <class T, int V, bool SUM, bool BACK, int PART, int U>
__global__ void __launch_bounds__(THREADS, blocks_of(V, BACK, PART)) scan_kernel(Args<T> a) {
    pdl_launch();
    const int64_t index = (int64_t)blockIdx.x * THREADS + threadIdx.x;
    const int order = (int)(index / a.lanes);
    if (order >= a.chunks) return;
    // the walk goes over the chunks from the side that the reduction read last
    const int chunk = PART == 1 ? a.chunks - 1 - order : order;
    const int64_t lane = index - order * a.lanes, per = a.D / V, b = lane / per, d = (lane - b * per) * V, c = b * a.D + d, C = a.B * a.D;
    // step i of the chunk in the direction of the recurrence is time first + i or first - i
    const int64_t from = chunk * a.size, first = BACK ? a.T_ - 1 - from : from;
    const int n = (int)min(a.T_ - from, a.size);
    constexpr int SIGN = BACK ? -1 : 1;
    Walk<T, V, SUM, BACK, PART> w;
    w.x = a.x.p + first * a.x.st + b * a.x.sb + d, w.sx = SIGN * a.x.st;
    w.gate = a.gate.p + first * a.gate.st + b * a.gate.sb + d, w.sgate = SIGN * a.gate.st;
    if constexpr (BACK) {
        w.dy = a.dy.p + first * a.dy.st + b * a.dy.sb + d, w.sdy = -a.dy.st;
        w.y = a.y.p + (first - 1) * a.y.st + b * a.y.sb + d, w.sy = -a.y.st;
        w.dgate = a.dgate + first * C + c;
    }
    w.out = a.out + first * C + c, w.sout = SIGN * C;
    float s[V], prod[V];
    int power[V];  // (sum form)
    // Resets: where a warp has one sequence and one chunk its lanes look at 32 steps at a time.
    const bool shared = a.reset && a.lanes % 32 == 0 && per % 32 == 0;
    const uint8_t *reset = a.reset ? a.reset + b * a.reset_b + (first + (shared ? SIGN * (int)(threadIdx.x & 31) : 0)) * a.reset_t : nullptr;
    const int64_t sreset = SIGN * (shared ? 32 : 1) * a.reset_t;
    int looked = 0;  // steps whose flags have been asked for
    uint32_t window = 0;
    uint8_t ahead = 0;
    const auto look = [&] {
        ahead = looked + (int)(threadIdx.x & 31) < n ? *reset : 0;
        reset += sreset;
        looked += 32;
    };
    if (shared) look();
    const auto cuts_of = [&](int i, int count) -> uint32_t {  // bit u: a reset at step i + u
        if (!a.reset) return 0;
        uint32_t bits = 0;
        if (shared) {
            if (i % 32 == 0) {
                window = __ballot_sync(0xffffffffu, ahead);
                if (looked < n) look();
            }
            return window >> (i % 32);
        }
#pragma unroll
        for (int u = 0; u < U; u++)
            if (u < count) {
                bits |= *reset ? 1u << u : 0u;
                reset += sreset;
            }
        return bits;
    };
    const auto advance = [&](const Step<T, V> &o, bool cut, bool earliest) {
        float r[V], dg[V];
#pragma unroll
        for (int v = 0; v < V; v++) {
            const float g = o.gate.get(v);
            float2 f;
            if constexpr (SUM)
                f = make_float2(expf(g), 1.f);
            else
                f = gates(g);
            if constexpr (!BACK) {
                const float in = SUM ? o.x.get(v) : f.y * o.x.get(v);
                s[v] = cut ? in : fmaf(f.x, s[v], in);
                r[v] = s[v];
            } else {
                const float D = o.dy.get(v) + s[v];
                if constexpr (PART == 1) {
                    float h = earliest ? (a.h0 ? a.h0[c + v] : 0.f) : o.y.get(v);
                    if (cut) h = 0.f;
                    const float into = SUM ? D : D * f.y;
                    r[v] = into;
                    dg[v] = SUM ? into * h * f.x : into * (h - o.x.get(v)) * f.x;
                }
                s[v] = cut ? 0.f : f.x * D;
            }
            if constexpr (PART == 0) {
                if constexpr (SUM) take_power(f.x, power[v]);
                prod[v] = cut || prod[v] < 0.f ? CUT : prod[v] * f.x;
            }
        }
        if constexpr (PART == 1) {
            Raw<T, V>::store(w.out, r);
            w.out += w.sout;
            if constexpr (BACK) {
                Raw<T, V>::store(w.dgate, dg);
                w.dgate += w.sout;
            }
        }
    };
    const auto normalise = [&] {  // after U steps at most: below 2^(U + 1) till then
        if constexpr (PART == 0 && SUM) {
#pragma unroll
            for (int v = 0; v < V; v++) {
                take_power(prod[v], power[v]);
                power[v] = max(-MOST_POWER, min(MOST_POWER, power[v]));
            }
        }
    };
    // Groups of U steps, the next one's loads under way during a group's arithmetic. The earliest step of the
    // time has no y before it: backward it is left to the single steps that follow.
    constexpr bool BEFORE = BACK && PART == 1;
    const int groups = (n - (BEFORE && first - (n - 1) == 0 ? 1 : 0)) / U;
    Step<T, V> p[U], q[U];
    uint32_t cp, cq;
    const auto fetch = [&](Step<T, V>(&to)[U], int group) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            w.load(to[u]);
            if constexpr (BEFORE) w.load_before(to[u]);
        }
        return cuts_of(group * U, U);
    };
    const auto compute = [&](const Step<T, V>(&of)[U], uint32_t cuts) {
#pragma unroll
        for (int u = 0; u < U; u++) advance(of[u], cuts >> u & 1, false);
        normalise();
    };
    if (groups) cp = fetch(p, 0);
    // The launches before this one read what it has read so far, and wrote none of it (the first of them began when all
    // earlier work was done): its first loads are under way before the states are there.
    pdl_wait();
#pragma unroll
    for (int v = 0; v < V; v++) {
        prod[v] = 1.f;
        power[v] = 0;
        s[v] = 0.f;
        if constexpr (PART == 1) s[v] = a.chunks > 1 ? a.carry[chunk * C + c + v].x : a.start ? a.start[c + v] : 0.f;
    }
    for (int k = 0; k < groups; k += 2) {
        if (k + 1 < groups) cq = fetch(q, k + 1);
        compute(p, cp);
        if (k + 1 < groups) {
            if (k + 2 < groups) cp = fetch(p, k + 2);
            compute(q, cq);
        }
    }
#pragma unroll 1
    for (int i = groups * U; i < n; i++) {
        w.load(p[0]);
        const bool earliest = BEFORE && i == n - 1 && first == n - 1;
        if (BEFORE && !earliest) w.load_before(p[0]);
        advance(p[0], cuts_of(i, 1) & 1, earliest);
        normalise();
    }
#pragma unroll
    for (int v = 0; v < V; v++) {
        if constexpr (PART == 0) {
            a.carry[chunk * C + c + v] = make_float2(prod[v], s[v]);
            if constexpr (SUM) a.power[chunk * C + c + v] = power[v];
        } else if (a.last && chunk == a.chunks - 1)
            a.last[c + v] = s[v];
    }
}

// The map of a piece of the time: s -> p 2^power s + q.
template <bool SUM> struct Map {
    float p = 1.f, q = 0.f;
    int power = 0;  // (0 in the average form)
};
// Of a state through it: the power first, which a state of 0 bears whatever it is.
template <bool SUM> __device__ __forceinline__ float through(const Map<SUM> &map, float s) {
    return map.p < 0.f ? map.q : fmaf(map.p, SUM ? scalbnf(s, map.power) : s, map.q);
}
// Of one piece and then another.
template <bool SUM> __device__ __forceinline__ Map<SUM> after(const Map<SUM> &first, const Map<SUM> &then) {
    Map<SUM> both;
    both.p = first.p < 0.f || then.p < 0.f ? CUT : first.p * then.p;
    both.q = through(then, first.q);
    if (SUM) both.power = first.power + then.power;
    return both;
}
// After up to 16 joins of normalised ones.
__device__ __forceinline__ void normalise(Map<true> &m) {
    take_power(m.p, m.power);
    m.power = max(-MOST_POWER, min(MOST_POWER, m.power));
}
__device__ __forceinline__ void normalise(Map<false> &) {}

// The state before every chunk, in place of its (P, Q): eight channels a block, the chunks divided between 128
// threads for each, which hold theirs and join them by doubling. (A warp for each of 32 runs of chunks, reading
// them twice, took 26 us for 2,048 chunks of 256 channels: the latency of its loads.)
template <bool SUM>
__global__ void __launch_bounds__(CARRY_RUNS * CARRY_CHANNELS) carry_kernel(float2 *carry, const int *power, const float *start, int64_t C, int chunks) {
    pdl_launch();
    pdl_wait();
    __shared__ float2 sums[CARRY_RUNS][CARRY_CHANNELS];
    __shared__ int powers[SUM ? CARRY_RUNS : 1][CARRY_CHANNELS];
    const int run = threadIdx.x / CARRY_CHANNELS, lane = threadIdx.x % CARRY_CHANNELS;
    const int64_t c = (int64_t)blockIdx.x * CARRY_CHANNELS + lane;
    const int each = (chunks + CARRY_RUNS - 1) / CARRY_RUNS, lo = run * each;
    Map<SUM> m[CARRY_EACH];
#pragma unroll
    for (int k = 0; k < CARRY_EACH; k++)
        if (k < each && lo + k < chunks && c < C) {
            const float2 of = carry[(lo + k) * C + c];
            m[k].p = of.x, m[k].q = of.y;
            if constexpr (SUM) m[k].power = power[(lo + k) * C + c];
        }
    Map<SUM> all = m[0];
#pragma unroll
    for (int k = 1; k < CARRY_EACH; k++) all = after(all, m[k]);
    normalise(all);
    const auto put = [&] {
        sums[run][lane] = make_float2(all.p, all.q);
        if constexpr (SUM) powers[run][lane] = all.power;
    };
    const auto get = [&](int r) {
        Map<SUM> of;
        of.p = sums[r][lane].x, of.q = sums[r][lane].y;
        if constexpr (SUM) of.power = powers[r][lane];
        return of;
    };
    put();
    __syncthreads();
#pragma unroll
    for (int d = 1; d < CARRY_RUNS; d *= 2) {
        Map<SUM> before;
        if (run >= d) before = get(run - d);
        __syncthreads();
        all = after(before, all);
        normalise(all);
        put();
        __syncthreads();
    }
    float s = start && c < C ? start[c] : 0.f;
    if (run) s = through(get(run - 1), s);
#pragma unroll
    for (int k = 0; k < CARRY_EACH; k++)
        if (k < each && lo + k < chunks && c < C) {
            carry[(lo + k) * C + c].x = s;
            s = through(m[k], s);
        }
}

// Chunks that the time is cut into: as many as make one wave of threads, each with 32 steps at least. 1 where that
// would be two: a third of a wave that reads once is as fast as a whole one that reads twice.
static int chunks_of(int64_t T, int64_t lanes, int blocks) {
    const int64_t want = (int64_t)SMS * THREADS * blocks / (lanes < 1 ? 1 : lanes), most = (T + 31) / 32;
    const int64_t n = want < 3 ? 1 : want < most ? want : most;
    return (int)(n < 1 ? 1 : n < MOST_CHUNKS ? n : MOST_CHUNKS);
}

template <class T, int V, bool SUM, bool BACK> static int run(Args<T> &a, cudaStream_t s) {
    constexpr int U = 4;
    a.lanes = a.B * a.D / V;
    a.chunks = chunks_of(a.T_, a.lanes, blocks_of(V, BACK, 1));
    a.size = (a.T_ + a.chunks - 1) / a.chunks;
    a.chunks = (int)((a.T_ + a.size - 1) / a.size);
    if (a.size > INT32_MAX) return D1_ERR_TOO_LARGE;
    if (a.chunks > 1 && !a.carry) return D1_ERR_BAD_ARGUMENT;
    a.power = (int *)(a.carry + a.chunks * a.B * a.D);
    const int64_t blocks = (a.lanes * a.chunks + THREADS - 1) / THREADS;
    if (blocks > INT32_MAX) return D1_ERR_TOO_LARGE;
    cudaLaunchAttribute attr;
    cudaLaunchConfig_t cfg = pdl_config(dim3((unsigned)blocks), dim3(THREADS), 0, s, &attr);
    cfg.numAttrs = 0;
    if (a.chunks > 1) {
        if (cudaError_t e = cudaLaunchKernelEx(&cfg, scan_kernel<T, V, SUM, BACK, 0, U>, a)) return (int)e;
        cfg.numAttrs = 1;
        cudaLaunchConfig_t mid = cfg;
        const int64_t C = a.B * a.D;
        mid.gridDim = dim3((unsigned)((C + CARRY_CHANNELS - 1) / CARRY_CHANNELS));
        mid.blockDim = dim3(CARRY_RUNS * CARRY_CHANNELS);
        if (cudaError_t e = cudaLaunchKernelEx(&mid, carry_kernel<SUM>, a.carry, a.power, a.start, C, a.chunks)) return (int)e;
    }
    return (int)cudaLaunchKernelEx(&cfg, scan_kernel<T, V, SUM, BACK, 1, U>, a);
}

template <class T> static bool vectors(const Span<const T> &s) {
    return aligned_to(8, s.p) && s.st % (8 / (int)sizeof(T)) == 0 && s.sb % (8 / (int)sizeof(T)) == 0;
}

template <class T, bool BACK> static int any(Args<T> a, int form, void *work, cudaStream_t s) {
    constexpr int V = 8 / sizeof(T);
    a.carry = (float2 *)work;
    if (!aligned_to(8, work)) return D1_ERR_BAD_ARGUMENT;
    const bool wide = a.D % V == 0 && vectors(a.gate) && vectors(a.x) && aligned_to(8, a.out) &&
                      (!BACK || (vectors(a.dy) && vectors(a.y) && aligned_to(8, a.dgate)));
    if (form == D1_SCAN_SUM) return wide ? run<T, V, true, BACK>(a, s) : run<T, 1, true, BACK>(a, s);
    return wide ? run<T, V, false, BACK>(a, s) : run<T, 1, false, BACK>(a, s);
}

// Whether sizes are in range: D, B, T >= 0 and all offsets of contiguous tensors within 62 bits.
static bool shape_ok(int64_t T, int64_t B, int64_t D) {
    return T >= 0 && B >= 0 && D >= 1 && T <= ((int64_t)1 << 40) && B <= ((int64_t)1 << 40) && D <= INT32_MAX &&
           (B == 0 || D <= ((int64_t)1 << 42) / B) && (T == 0 || B * D <= ((int64_t)1 << 58) / T);
}

// Whether the strides of a [T, B, D] operand are: its last element lies within 60 bits of its first.
static bool strides_ok(int64_t st, int64_t sb, int64_t T, int64_t B) {
    constexpr int64_t MOST = (int64_t)1 << 59;
    return st >= 0 && sb >= 0 && st <= MOST / (T < 2 ? 1 : T - 1) && sb <= MOST / (B < 2 ? 1 : B - 1);
}
// The bytes from the first to the last that an operand (or a result) has.
struct Range {
    uintptr_t from, to;
};
static Range range_of(const void *p, int64_t st, int64_t sb, int64_t T, int64_t B, int64_t D, int size) {
    const uintptr_t at = (uintptr_t)p;
    return {at, p && T > 0 && B > 0 ? at + (uintptr_t)(((T - 1) * st + (B - 1) * sb + D) * size) : at};
}
static Range range_of(const void *p, int64_t count, int size) { return range_of(p, 0, 0, 1, 1, count, size); }
static bool meet(const Range &a, const Range &b) { return a.from < b.to && b.from < a.to && a.from < a.to && b.from < b.to; }
static bool meet_any(const Range &a, std::initializer_list<Range> others) {
    for (const Range &b : others)
        if (meet(a, b)) return true;
    return false;
}

}  // namespace gs
}  // namespace d1

extern "C" int64_t d1_gated_scan_work_bytes(int64_t T, int64_t B, int64_t D) {
    using namespace d1::gs;
    if (!shape_ok(T, B, D)) return -1;
    // of any width, direction and type
    int64_t most = 0;
    for (const int V : {1, 2, 4})
        for (const bool back : {false, true}) {
            const int chunks = chunks_of(T, B * D / V, blocks_of(V, back, 1));
            if (chunks > 1 && chunks > most) most = chunks;
        }
    return 8 * ((3 * most + 1) / 2) * B * D;  // 8 bytes of (P, Q) and 4 of a power
}

extern "C" int d1_gated_scan(const void *x, int64_t x_t, int64_t x_b, const void *gate, int64_t gate_t, int64_t gate_b,
                             int type, int form, int64_t T, int64_t B, int64_t D, const float *h0, const uint8_t *reset,
                             int64_t reset_t, int64_t reset_b, void *y, float *last, void *work, void *stream) {
    using namespace d1;
    if (!type_ok(type) || (form != D1_SCAN_AVERAGE && form != D1_SCAN_SUM) || !gs::shape_ok(T, B, D) ||
        (T && B && (!x || !gate || !y)) || !gs::strides_ok(x_t, x_b, T, B) || !gs::strides_ok(gate_t, gate_b, T, B) ||
        !gs::strides_ok(reset_t, reset_b, T, B) || !element_aligned(x, type) || !element_aligned(gate, type) || !element_aligned(y, type) || !aligned_to(4, h0, last))
        return D1_ERR_BAD_ARGUMENT;
    const int size = type == D1_TYPE_F32 ? 4 : 2;
    const gs::Range xs = gs::range_of(x, x_t, x_b, T, B, D, size), gates = gs::range_of(gate, gate_t, gate_b, T, B, D, size),
                    resets = gs::range_of(reset, reset_t, reset_b, T, B, 1, 1), ys = gs::range_of(y, T * B * D, size),
                    h0s = gs::range_of(h0, B * D, 4), lasts = gs::range_of(last, B * D, 4);
    if (gs::meet_any(ys, {xs, gates, resets, h0s, lasts}) || gs::meet_any(lasts, {xs, gates, resets}) || (last != h0 && gs::meet(lasts, h0s)))
        return D1_ERR_BAD_ARGUMENT;
    const cudaStream_t s = (cudaStream_t)stream;
    if (B == 0) return 0;
    if (T == 0) {  // the state is what it was
        if (!last || last == h0) return 0;
        return (int)(h0 ? cudaMemcpyAsync(last, h0, (size_t)(B * D) * 4, cudaMemcpyDeviceToDevice, s)
                        : cudaMemsetAsync(last, 0, (size_t)(B * D) * 4, s));
    }
    const auto go = [&](auto one) {
        using E = decltype(one);
        gs::Args<E> a{};
        a.x = {(const E *)x, x_t, x_b};
        a.gate = {(const E *)gate, gate_t, gate_b};
        a.out = (E *)y;
        a.reset = reset, a.reset_t = reset_t, a.reset_b = reset_b;
        a.start = h0, a.last = last;
        a.T_ = T, a.B = B, a.D = D;
        return gs::any<E, false>(a, form, work, s);
    };
    return type == D1_TYPE_F32 ? go(float{}) : type == D1_TYPE_BF16 ? go(__nv_bfloat16{}) : go(__half{});
}

extern "C" int d1_gated_scan_backward(const void *dy, int64_t dy_t, int64_t dy_b, const void *x, int64_t x_t, int64_t x_b,
                                      const void *gate, int64_t gate_t, int64_t gate_b, const void *y, int64_t y_t,
                                      int64_t y_b, int type, int form, int64_t T, int64_t B, int64_t D, const float *h0,
                                      const float *dlast, const uint8_t *reset, int64_t reset_t, int64_t reset_b, void *dx,
                                      void *dgate, float *dh0, void *work, void *stream) {
    using namespace d1;
    if (!type_ok(type) || (form != D1_SCAN_AVERAGE && form != D1_SCAN_SUM) || !gs::shape_ok(T, B, D) ||
        (T && B && (!dy || !x || !gate || !y || !dx || !dgate)) || !gs::strides_ok(x_t, x_b, T, B) ||
        !gs::strides_ok(gate_t, gate_b, T, B) || !gs::strides_ok(y_t, y_b, T, B) || !gs::strides_ok(dy_t, dy_b, T, B) ||
        !gs::strides_ok(reset_t, reset_b, T, B) ||
        !element_aligned(x, type) || !element_aligned(gate, type) || !element_aligned(y, type) ||
        !element_aligned(dy, type) || !element_aligned(dx, type) || !element_aligned(dgate, type) ||
        !aligned_to(4, h0, dlast, dh0))
        return D1_ERR_BAD_ARGUMENT;
    const int size = type == D1_TYPE_F32 ? 4 : 2;
    const gs::Range xs = gs::range_of(x, x_t, x_b, T, B, D, size), gates = gs::range_of(gate, gate_t, gate_b, T, B, D, size),
                    ys = gs::range_of(y, y_t, y_b, T, B, D, size), dys = gs::range_of(dy, dy_t, dy_b, T, B, D, size),
                    resets = gs::range_of(reset, reset_t, reset_b, T, B, 1, 1), h0s = gs::range_of(h0, B * D, 4), dlasts = gs::range_of(dlast, B * D, 4),
                    dxs = gs::range_of(dx, T * B * D, size), dgates = gs::range_of(dgate, T * B * D, size), dh0s = gs::range_of(dh0, B * D, 4);
    for (const gs::Range &q : {dxs, dgates})
        if (gs::meet_any(q, {xs, gates, ys, dys, resets, h0s, dlasts, dh0s})) return D1_ERR_BAD_ARGUMENT;
    if (gs::meet(dxs, dgates) || gs::meet_any(dh0s, {xs, gates, ys, dys, resets, h0s}) || (dh0 != dlast && gs::meet(dh0s, dlasts)))
        return D1_ERR_BAD_ARGUMENT;
    const cudaStream_t s = (cudaStream_t)stream;
    if (B == 0) return 0;
    if (T == 0) {
        if (!dh0 || dh0 == dlast) return 0;
        return (int)(dlast ? cudaMemcpyAsync(dh0, dlast, (size_t)(B * D) * 4, cudaMemcpyDeviceToDevice, s)
                           : cudaMemsetAsync(dh0, 0, (size_t)(B * D) * 4, s));
    }
    const auto go = [&](auto one) {
        using E = decltype(one);
        gs::Args<E> a{};
        a.x = {(const E *)x, x_t, x_b};
        a.gate = {(const E *)gate, gate_t, gate_b};
        a.y = {(const E *)y, y_t, y_b};
        a.dy = {(const E *)dy, dy_t, dy_b};
        a.out = (E *)dx, a.dgate = (E *)dgate;
        a.reset = reset, a.reset_t = reset_t, a.reset_b = reset_b;
        a.start = dlast, a.h0 = h0, a.last = dh0;
        a.T_ = T, a.B = B, a.D = D;
        return gs::any<E, true>(a, form, work, s);
    };
    return type == D1_TYPE_F32 ? go(float{}) : type == D1_TYPE_BF16 ? go(__nv_bfloat16{}) : go(__half{});
}
