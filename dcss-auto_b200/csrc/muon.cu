// Muon: momentum, orthogonalisation of the update by Newton-Schulz products, and
// the step, over many weight matrices at a time (sm_100a, tcgen05 + TMA).
//
//   m' = mu m + g        u = g + mu m' (Nesterov) or m'
//   X = u / |u|_F, then `steps` times:  A = X X^T (or X^T X)   F = a I + b A + c A^2   X' = F X (or X F)
//   p' = p (1 - lr decay) - lr 0.2 sqrt(max(rows, cols)) X
//
// with the published coefficients (a, b, c) = (3.4445, -4.7750, 2.0315), which bring
// every singular value of X between about 0.7 and 1.2.
//
// Rounding. The products run on the tensor cores in fp16 with fp32 sums: X, A and F are bounded (by 1.3, 1.7 and 3.5),
// so that a scale of 2^12 keeps all of them inside fp16's range, and fp16 has eight times bf16's precision at the same
// rate. Singular directions that the update hardly has are amplified by a = 3.4 a step, 485 in five, and with them
// whatever rounding puts there: of a gradient of low rank the result would be noise to a large part (simulated, rank 32 of
// 512: 3 % of its norm in fp16, 22 % in bf16). So X is held as a pair hi + lo of fp16, 22 bits, and X' = F hi + a lo: where X
// has nothing F is a, and the pair is carried on as one; elsewhere F lo is not a lo, an error of hi's size, but
// in directions that X has (0.16 % there, 0.2 % of a full-rank one). That is a bf16 result's own rounding (0.17 %), but eight times an
// fp16 one's: where the caller asks for it (`precise`), A and F are pairs too and a product takes all three terms, as good as one in
// fp32 for up to three times the products' time (8,192 x 8,192 28.6 ms in place of 10.0, 7 x 1,777 x 1,003 770 us in place of 371, 512 x 512 182
// in place of 123, the conv policy's six 224 in place of 145). So it is in a matrix with a side of at most 64, where few
// roundings average out (up to 1 % in some), and where its time is the launches' all the same. Where all matrices are as narrow as that up to five
// steps are taken another way (muon_narrow.cuh).
//
// The three products of all matrices are one launch each. A and F are symmetric: only the tiles on and below the
// diagonal are computed and stored, and read transposed for those above. The epilogues hold the rest of the
// formulas, the last one the step itself. All operands are blocks of 64 x 64 elements (d1_muon.h) that the TMA
// swizzles on its way to shared memory, as K-major operands or as MN-major ones: X is never transposed.
//
// Measured (one B200). 8,192 x 8,192 bf16: 10.0 ms, 1.3 PFLOP/s while the products run (a library product sustains 1.38
// under the power limit). 72 matrices of 12 layers of 1,024, with masters, momentum and copies: 3.89 ms (floor 1.64). The conv policy's six:
// 145 us, 17 launches. A pair of CTAs takes 0.43 us for a block of 64 of the sum of its 256 x 256 tile: 32 KB into shared memory and 48 KB read
// for 512 cycles of the tensor pipe, 640 cycles at 128 bytes each, which bound it.
#include <cuda.h>
#include <math.h>

#include <algorithm>
#include <atomic>
#include <new>
#include <type_traits>

#include "d1_common.cuh"
#include "d1_elem.cuh"
#include "d1_muon.h"
#include "d1_pdl.cuh"
#include "d1_rows.h"
#include "tc_ptx.cuh"

namespace d1 {
namespace muon {

using namespace tcx;

constexpr int SMS = 148, STAGES = 5, HALF_BYTES = 2 * BLOCK_BYTES, STAGE_BYTES = 2 * HALF_BYTES, EPI_WARPS = 8;
constexpr int THREADS = 64 + 32 * EPI_WARPS, PREP = 256;
constexpr int ROOM = BLOCK_BYTES / 2;  // 32 x 32 elements of two operands; an epilogue warp has two
constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + EPI_WARPS * 2 * ROOM + 1024 + 512;
constexpr uint32_t WAIT_LIMIT = 1u << 22;
constexpr float SCALE = 4096.f, UNSCALE = 1.f / 4096.f;  // of X, A and F in fp16
constexpr float NS_A = 3.4445f, NS_B = -4.7750f, NS_C = 2.0315f;

// The last wait that ran out, on this device. While it stands no step changes a master: some of what it is made from is missing.
__device__ int g_error;
// The same in pinned host memory, of any device, where the caller sees it without a synchronisation (NULL: nowhere).
static std::atomic<int *> told{nullptr};

struct Job {
    const Matrix *matrices;  // NULL: a stack of `one`
    const Tile *symmetric, *full;
    const Part *parts;
    Matrix one;
    int64_t grad_step, out_step;  // bytes from one matrix of the stack to the next
    int block_step;
    int count_symmetric, count_full, per_symmetric, per_full, tm, tn;
    uint8_t *work;
    double *partials;
    float mu;
    int nesterov;
    double lr;
    int from;   // which hi is read
    int steps;
    int adders;  // narrow matrices: blocks that add the sums of one
    int *told;
};

__device__ __forceinline__ void fail(const Job &o, int code) {
    atomicExch(&g_error, code);
    if (o.told) {
        *(volatile int *)o.told = code;
        __threadfence_system();
    }
}

__device__ __forceinline__ Matrix matrix_of(const Job &o, int m) {
    if (o.matrices) return o.matrices[m];
    Matrix x = o.one;
    x.grad = (const char *)x.grad + m * o.grad_step;
    x.out = (char *)x.out + m * o.out_step;
    const int b = m * o.block_step;
    x.hi[0] += b, x.hi[1] += b, x.lo += b, x.lo2 += b, x.gram += b, x.quad += b;
    x.part0 += m * x.parts;
    return x;
}
__device__ __forceinline__ Tile tile_of(const Job &o, bool symmetric, int t) {
    if (o.matrices) return symmetric ? o.symmetric[t] : o.full[t];
    const int per = symmetric ? o.per_symmetric : o.per_full;
    Tile r;
    r.matrix = t / per;
    int i, j;
    if (symmetric)
        symmetric_tile(t - r.matrix * per, i, j);
    else
        grouped_tile(t - r.matrix * per, o.tm, o.tn, i, j);
    r.i = (uint16_t)i, r.j = (uint16_t)j;
    return r;
}

// A role's tiles first, first + step, ..., each looked up while the one before it is worked on: its record two tiles
// ahead, its matrix one, so that no load is waited for (a lookup in place took a microsecond of each tile's time).
struct Tiles {
    const Job &o;
    const bool symmetric;
    const int count, step;
    int at;
    Tile next, next2;
    Matrix next_m;

    __device__ __forceinline__ Tiles(const Job &o, bool symmetric, int count, int first, int step) : o(o), symmetric(symmetric), count(count), step(step), at(first) {
        next = tile_of(o, symmetric, at);
        next2 = at + step < count ? tile_of(o, symmetric, at + step) : next;
        next_m = matrix_of(o, next.matrix);
    }
    // The next tile to work on and its matrix; false when there is none.
    __device__ __forceinline__ bool take(Matrix &m, Tile &tile) {
        if (at >= count) return false;
        tile = next, m = next_m;
        next = next2;
        at += step;
        if (at < count) next_m = matrix_of(o, next.matrix);
        if (at + step < count) next2 = tile_of(o, symmetric, at + step);
        return true;
    }
};

// The tiles first, first + step, ... of one matrix.
struct MatrixTiles {
    const Matrix &matrix;
    const bool symmetric;
    int at, step, count, tm, tn;

    __device__ __forceinline__ MatrixTiles(const Matrix &m, bool symmetric, int first, int step) : matrix(m), symmetric(symmetric), at(first), step(step) {
        tm = tiles_of(symmetric ? m.sb : m.rb, 2), tn = tiles_of(symmetric ? m.sb : m.cb, 2);
        count = symmetric ? tm * (tm + 1) / 2 : tm * tn;
    }
    __device__ __forceinline__ bool take(Matrix &m, Tile &tile) {
        if (at >= count) return false;
        int i, j;
        if (symmetric)
            symmetric_tile(at, i, j);
        else
            grouped_tile(at, tm, tn, i, j);
        m = matrix, tile.matrix = 0, tile.i = (uint16_t)i, tile.j = (uint16_t)j;
        at += step;
        return true;
    }
};

// ---------------------------------------------------------------- momentum, norm, X

// n of 8 consecutive elements (the others 0).
template <class T> __device__ __forceinline__ void load8(const T *p, int n, bool wide, float (&v)[8]) {
    if (wide) {
        constexpr int N = 16 / sizeof(T);
#pragma unroll
        for (int k = 0; k < 8; k += N) {
            const Elems<T, N> e = *reinterpret_cast<const Elems<T, N> *>(p + k);
#pragma unroll
            for (int i = 0; i < N; i++) v[k + i] = to_f32(e.v[i]);
        }
    } else
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = k < n ? to_f32(p[k]) : 0.f;
}
__device__ __forceinline__ void load8(const void *base, int type, int64_t at, int n, float (&v)[8]) {
    if (type == D1_TYPE_F32) {
        const float *p = (const float *)base + at;
        load8(p, n, n == 8 && ((uintptr_t)p & 15) == 0, v);
    } else if (type == D1_TYPE_BF16) {
        const __nv_bfloat16 *p = (const __nv_bfloat16 *)base + at;
        load8(p, n, n == 8 && ((uintptr_t)p & 15) == 0, v);
    } else {
        const __half *p = (const __half *)base + at;
        load8(p, n, n == 8 && ((uintptr_t)p & 15) == 0, v);
    }
}

// Where 8 columns of a row stand in a block of lo that is no operand: as the epilogues take them, 32 x 32 elements
// after 32 x 32, of them 8 columns after 8, row after row (a lane has a row).
__device__ __forceinline__ int lo_at(int row, int col) { return ((row >> 5) * 2 + (col >> 5)) * ROOM / 2 + (col & 31) / 8 * 512 + (row & 31) * 16; }

// Sum over the block in a fixed order, in every thread.
__device__ __forceinline__ double block_sum(double s, double *shared) {
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = s;
    __syncthreads();
    s = 0.;
#pragma unroll
    for (int w = 0; w < PREP / 32; w++) s += shared[w];
    return s;
}

// u at n elements of row i from column j on, and the momentum, which UPDATE brings up to date.
template <bool UPDATE> __device__ __forceinline__ void momentum8(const Job &o, const Matrix &m, int i, int j, int n, float (&u)[8]) {
    load8(m.grad, m.grad_type, i * m.pitch + j, n, u);
    if (!m.momentum) return;
    float *p = m.momentum + (int64_t)i * m.cols + j, v[8];
    const bool wide = n == 8 && ((uintptr_t)p & 15) == 0;
    load8(p, n, wide, v);
    if (UPDATE) {
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = fmaf(o.mu, v[k], u[k]);
        if (wide) {
            *(float4 *)p = make_float4(v[0], v[1], v[2], v[3]);
            *(float4 *)(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
        } else
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (k < n) p[k] = v[k];
    }
#pragma unroll
    for (int k = 0; k < 8; k++) u[k] = o.nesterov ? fmaf(o.mu, v[k], u[k]) : v[k];
}

// FIRST: the new momentum and the sum of the squares of u (in fp64: squares of fp32 numbers neither overflow
// nor vanish there). Else X = u / |u|, as hi + lo.
template <bool FIRST> __global__ void __launch_bounds__(PREP) prepare_kernel(Job o) {
    __shared__ double shared[PREP / 32];
    pdl_launch();  // the next launch's blocks come in as these leave, and wait for the last of them
    pdl_wait();
    Part part;
    if (o.matrices)
        part = o.parts[blockIdx.x];
    else
        part.matrix = blockIdx.x / o.one.parts, part.k = blockIdx.x % o.one.parts;
    const Matrix m = matrix_of(o, part.matrix);
    double sum = 0., inverse = 0.;
    if (!FIRST) {
        if ((int)threadIdx.x < m.parts) sum = o.partials[m.part0 + threadIdx.x];
        const double norm = sqrt(block_sum(sum, shared));
        inverse = norm == 0. ? 0. : (double)SCALE / norm;
    }
    for (int b = part.k; b < m.rb * m.cb; b += m.parts) {
        const int ib = b / m.cb, jb = b - ib * m.cb;
#pragma unroll
        for (int q = 0; q < 2; q++) {
            const int e = threadIdx.x + PREP * q, row = e >> 3, col = (e & 7) * 8;
            const int i = ib * SIDE + row, j = jb * SIDE + col, n = i < m.rows ? min(8, max(0, m.cols - j)) : 0;
            float u[8] = {};
            if (n) momentum8<FIRST>(o, m, i, j, n, u);
            if (FIRST) {
#pragma unroll
                for (int k = 0; k < 8; k++) sum = fma((double)u[k], (double)u[k], sum);
            } else {
                Elems<__half, 8> hi, lo;
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const float x = (float)((double)u[k] * inverse);
                    hi.v[k] = __float2half_rn(x);
                    lo.v[k] = __float2half_rn(x - __half2float(hi.v[k]));
                }
                const int at = row * 128 + col * 2;
                *reinterpret_cast<Elems<__half, 8> *>(o.work + (int64_t)(m.hi[0] + b) * BLOCK_BYTES + at) = hi;
                *reinterpret_cast<Elems<__half, 8> *>(o.work + (int64_t)(m.lo + b) * BLOCK_BYTES + (m.fine ? at : lo_at(row, col))) = lo;
            }
        }
    }
    if (FIRST) {
        sum = block_sum(sum, shared);
        if (threadIdx.x == 0) o.partials[m.part0 + part.k] = sum;
    }
}

// ---------------------------------------------------------------- products

enum Mode { SINGLES, PAIRS, SPLITS };  // a CTA, a pair of them, or a cluster for a tile
enum Phase { GRAM, QUAD, APPLY, STEP };  // A; F; X'; the step with the last X' (or the result itself)

// Where the operands of a phase lie: block (i, k) of the first at a + i * ai + k * ak, of the second at
// b + j * bj + k * bk; their blocks along i, j and k. A symmetric one (A, F) has the tiles on and below its diagonal: where k is
// past the tile, block (k, i) is taken, as an MN-major operand.
struct Operands {
    int a, ai, ak, b, bj, bk, ni, nj, nk;
    bool a_mn, b_mn, a_half, b_half;
    int terms;         // 1; 3 where operands are pairs: hi hi, lo hi, hi lo (lo lo is below fp32's last bit)
    int a_lo, b_lo;    // from a hi block to its lo block
};
__device__ __forceinline__ Operands operands(const Matrix &m, int phase, int from) {
    const int hi = from ? m.hi[1] : m.hi[0], x_lo = (from ? m.lo2 : m.lo) - hi, f_lo = m.sb * m.sb, terms = m.fine ? 3 : 1;
    if (phase == GRAM)
        return m.tall ? Operands{hi, 1, m.cb, hi, 1, m.cb, m.sb, m.sb, m.rb, true, true, false, false, terms, x_lo, x_lo}
                      : Operands{hi, m.cb, 1, hi, m.cb, 1, m.sb, m.sb, m.cb, false, false, false, false, terms, x_lo, x_lo};
    if (phase == QUAD) return Operands{m.gram, m.sb, 1, m.gram, m.sb, 1, m.sb, m.sb, m.sb, false, false, true, true, terms, f_lo, f_lo};
    return m.tall ? Operands{hi, m.cb, 1, m.quad, m.sb, 1, m.rb, m.cb, m.sb, false, false, false, true, terms, x_lo, f_lo}
                  : Operands{m.quad, m.sb, 1, hi, 1, m.cb, m.rb, m.cb, m.sb, false, true, true, false, terms, f_lo, x_lo};
}

// Where part r of `parts` of a product's sum begins.
__device__ __forceinline__ int part_of(const Operands &p, int r, int parts) { return p.nk * p.terms * r / parts; }

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t mapa(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The same for threads that come there one by one; all of the cluster's threads do.
__device__ __forceinline__ void cluster_meet() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// A TMA load into this CTA's shared memory that completes on a barrier of either CTA of the pair.
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void mma_pair(uint32_t tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// All but the last committed bulk store have finished reading shared memory.
__device__ __forceinline__ void bulk_wait_read_but_one() { asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory"); }
__device__ __forceinline__ void commit_pair(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// A warp's share of the epilogue is a row of the tile a lane, taken 32 columns at a time. Operands and results pass
// through shared memory of the warp's own, by TMA, two rooms in turn: a lane that reads or writes its row in memory
// touches a line of its own with each access, which bounded the epilogues (X' of 1024 x 1024 x 1024 at 0.66 PFLOP/s, the
// step with it at 0.33).
struct Halves8 {
    __half2 v[4];
};
__device__ __forceinline__ void unpack(uint4 w, float (&x)[8]) {
    const Halves8 h = *reinterpret_cast<const Halves8 *>(&w);
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const float2 f = __half22float2(h.v[k]);
        x[2 * k] = f.x, x[2 * k + 1] = f.y;
    }
}
// x as hi + lo.
__device__ __forceinline__ void split(const float (&x)[8], uint4 &hi, uint4 &lo) {
    Halves8 h, l;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        h.v[k] = __floats2half2_rn(x[2 * k], x[2 * k + 1]);
        const float2 f = __half22float2(h.v[k]);
        l.v[k] = __floats2half2_rn(x[2 * k] - f.x, x[2 * k + 1] - f.y);
    }
    hi = *reinterpret_cast<const uint4 *>(&h);
    lo = *reinterpret_cast<const uint4 *>(&l);
}

// Column j of row i of 32 in a room of 32 fp32 columns: pieces of 16 bytes at piece ^ (row & 7), so that neither rows nor
// columns meet in a bank.
__device__ __forceinline__ int place_of(int r, int c) { return r * 32 + ((((c >> 2) ^ (r & 7)) << 2) | (c & 3)); }

// The parameters of 32 rows and this lane's column, asked for ahead of the step on them.
__device__ __forceinline__ void load_params(const Matrix &m, int i0, int j0, float (&p)[32]) {
    const int j = j0 + (threadIdx.x & 31), rows = j < m.cols ? min(32, m.rows - i0) : 0;
    const float *at = m.param + (int64_t)i0 * m.cols + j;
#pragma unroll
    for (int r = 0; r < 32; r++, at += m.cols)
        if (r < rows) p[r] = *at;
}

// The step on 32 rows of 32 columns (or the result itself): x holds a row a lane, memory is touched a row at a time, the room turns
// one into the other.
__device__ __forceinline__ void finish(const Job &o, const Matrix &m, int i0, int j0, const float (&x)[32], const float (&p)[32], float *room) {
    const int lane = threadIdx.x & 31;
    __syncwarp();
#pragma unroll
    for (int k = 0; k < 32; k += 4) *reinterpret_cast<float4 *>(room + place_of(lane, k)) = make_float4(x[k], x[k + 1], x[k + 2], x[k + 3]);
    __syncwarp();
    const int rows = j0 + lane < m.cols ? min(32, m.rows - i0) : 0;
    int64_t at = (int64_t)i0 * m.cols + j0 + lane;
    float turned[32];  // all of them before the first store: the compiler keeps loads behind stores that might meet them
#pragma unroll
    for (int r = 0; r < 32; r++) turned[r] = room[place_of(r, lane)];
    if (!m.param) {
        const bool bf16 = m.out_type == D1_TYPE_BF16;
#pragma unroll
        for (int r = 0; r < 32; r++, at += m.cols)
            if (r < rows) {
                const float y = turned[r] * UNSCALE;
                if (bf16)
                    ((__nv_bfloat16 *)m.out)[at] = __float2bfloat16_rn(y);
                else
                    ((__half *)m.out)[at] = __float2half_rn(y);
            }
    } else {
        const float keep = (float)(1. - o.lr * (double)m.keep_decay), rate = (float)(-o.lr * (double)m.rate) * UNSCALE;
#pragma unroll
        for (int r = 0; r < 32; r++, at += m.cols)
            if (r < rows) {
                const float y = fmaf(rate, turned[r], p[r] * keep);
                m.param[at] = y;
                if (m.out) ((__nv_bfloat16 *)m.out)[at] = __float2bfloat16_rn(y);
            }
    }
    __syncwarp();
}

// A CTA's part in the products, role by role: warp 0 loads blocks of 64 x 64 elements, 128 rows of each operand a
// stage, through a ring of five; one thread of warp 1 (of a pair's first CTA) issues the products into one of two
// accumulators; eight warps read the other one, 128 rows of the tile in each CTA. Every role goes over the same tiles. The
// ring and the accumulators go on from one product to the next.
//
// A tile is 128 x 128 elements, or 256 x 256 of a PAIR. SPLIT: a cluster of 2, 4 or 8 CTAs takes a tile of 128 x 128 together, each
// a part of the sum. Each then owns some of the tile's sixteen units of 32 x 32: the others' parts of them come to its shared
// memory, and it adds them in the order of the parts. It is for products of few tiles with long sums: X X^T of 512 x 3136
// has ten, of 49 blocks each. Single products X' have too many tiles for it wherever their sums are long enough; those of pairs from 4 x 4 blocks on
// (189 of 100,000 shapes up to 200 x 600) are left whole too.
template <bool PAIR> struct Roles {
    static constexpr int SIDES = PAIR ? 4 : 2, COLS = SIDES * SIDE;  // blocks along a tile; columns of an accumulator

    const CUtensorMap &map, &map_units;
    const Job &o;
    uint8_t *const smem;
    const uint32_t full0, empty0, accf0, acce0, sides_at;
    uint32_t tmem;
    const int warp, lane, rank;
    int parts, part;          // of a divided sum
    int it = 0, in_flight = 0;  // stages that the role has gone through
    int local = 0;            // accumulators
    uint32_t turns = 0, pending = 0;  // of an epilogue warp's two rooms, a bit each: the parity of the next wait, a load that is under way
    bool ok = true;

    static __device__ __forceinline__ constexpr bool symmetric(int phase) { return phase == GRAM || phase == QUAD; }

    template <int PHASE, bool SPLIT, class List> __device__ __forceinline__ void load(List &list, int from) {
        Matrix m;
        Tile tile;
        while (ok && list.take(m, tile)) {
            const Operands p = operands(m, PHASE, from);
            const int i0 = tile.i * SIDES + 2 * rank, j0 = tile.j * SIDES + 2 * rank;
            // blocks that exist, of the tile (whose bytes the barrier expects) and of this CTA
            const int all = min(SIDES, p.ni - tile.i * SIDES) + min(SIDES, p.nj - tile.j * SIDES);
            const int na = min(2, p.ni - i0), nb = min(2, p.nj - j0);
            const int end = part_of(p, SPLIT ? part + 1 : 1, SPLIT ? parts : 1);
            for (int n = part_of(p, SPLIT ? part : 0, SPLIT ? parts : 1), k = n % p.nk, term = n / p.nk; n < end; n++, it++) {
                const int s = it % STAGES;
                const bool a_turned = p.a_half && k / SIDES > tile.i, b_turned = p.b_half && k / SIDES > tile.j;
                const int ai = a_turned ? p.ak : p.ai, ak = a_turned ? p.ai : p.ak, bj = b_turned ? p.bk : p.bj, bk = b_turned ? p.bj : p.bk;
                const int a_at = (p.a + i0 * ai + k * ak + (term == 1 ? p.a_lo : 0)) * SIDE, b_at = (p.b + j0 * bj + k * bk + (term == 2 ? p.b_lo : 0)) * SIDE;
                if (++k == p.nk) k = 0, term++;
                if (it >= STAGES && !mbar_wait(empty0 + 8 * s, ((uint32_t)(it / STAGES) & 1u) ^ 1u, WAIT_LIMIT)) {
                    ok = false;
                    break;
                }
                if (it >= STAGES) in_flight = it - STAGES + 1;
                const uint32_t a_dst = smem_u32(smem + s * STAGE_BYTES), b_dst = a_dst + HALF_BYTES;
                const uint32_t full = PAIR ? mapa(full0 + 8 * s, 0) : full0 + 8 * s;
                if (rank == 0) mbar_expect_tx(full0 + 8 * s, all * BLOCK_BYTES);
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    if (PAIR) {
                        if (h < na) tma_load_2d_pair(a_dst + h * BLOCK_BYTES, &map, full, 0, a_at + h * ai * SIDE);
                        if (h < nb) tma_load_2d_pair(b_dst + h * BLOCK_BYTES, &map, full, 0, b_at + h * bj * SIDE);
                    } else {
                        if (h < na) tma_load_2d(a_dst + h * BLOCK_BYTES, &map, full, 0, a_at + h * ai * SIDE);
                        if (h < nb) tma_load_2d(b_dst + h * BLOCK_BYTES, &map, full, 0, b_at + h * bj * SIDE);
                    }
                }
            }
        }
    }
    // After the last product: what is under way lands before the block leaves.
    __device__ __forceinline__ void loaded() {
        if (!ok) {
            fail(o, 1);
            if (rank == 0)  // copies under way land before the block leaves
                for (int i = in_flight; i < it; i++) mbar_wait(full0 + 8 * (i % STAGES), (uint32_t)(i / STAGES) & 1u, WAIT_LIMIT);
        } else  // and so do the last signals that a stage is free
            for (int i = it > STAGES ? it - STAGES : 0; i < it; i++)
                mbar_wait(empty0 + 8 * (i % STAGES), (uint32_t)(i / STAGES) & 1u, WAIT_LIMIT);
    }

    template <int PHASE, bool SPLIT, class List> __device__ __forceinline__ void multiply(List &list, int from) {
        Matrix m;
        Tile tile;
        for (; ok && list.take(m, tile); local++) {
            const Operands p = operands(m, PHASE, from);
            constexpr uint32_t BASE = (1u << 4) | ((uint32_t)(COLS >> 3) << 17) | ((uint32_t)(COLS >> 4) << 24);  // fp16, fp32 sums
            const int b = local & 1;
            const uint32_t acc = tmem + (uint32_t)(b * COLS);
            if (local >= 2 && !mbar_wait(acce0 + 8 * b, ((uint32_t)(local >> 1) & 1u) ^ 1u, WAIT_LIMIT)) {
                fail(o, 2);
                ok = false;
                break;
            }
            tc_fence_after();
            const int begin = part_of(p, SPLIT ? part : 0, SPLIT ? parts : 1), end = part_of(p, SPLIT ? part + 1 : 1, SPLIT ? parts : 1);
            for (int n = begin, k = begin % p.nk; n < end; n++, it++) {
                const int s = it % STAGES;
                if (!mbar_wait(full0 + 8 * s, (uint32_t)(it / STAGES) & 1u, WAIT_LIMIT)) {
                    fail(o, 3);
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t a = smem_u32(smem + s * STAGE_BYTES), c = a + HALF_BYTES;
                const bool a_mn = p.a_mn || (p.a_half && k / SIDES > tile.i), b_mn = p.b_mn || (p.b_half && k / SIDES > tile.j);
                const uint32_t idesc = BASE | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u);
                if (++k == p.nk) k = 0;
#pragma unroll
                for (int kk = 0; kk < SIDE / 16; kk++) {
                    const uint64_t da = a_mn ? desc_sw128_mn(a + kk * 2048, BLOCK_BYTES) : desc_sw128_k(a + kk * 32);
                    const uint64_t db = b_mn ? desc_sw128_mn(c + kk * 2048, BLOCK_BYTES) : desc_sw128_k(c + kk * 32);
                    if (PAIR)
                        mma_pair(acc, da, db, idesc, n > begin || kk);
                    else
                        mma_bf16(acc, da, db, idesc, n > begin || kk);
                }
                if (PAIR) {
                    commit_pair(empty0 + 8 * s);
                    commit_pair(mapa(empty0 + 8 * s, 1));
                } else
                    mma_commit(empty0 + 8 * s);
            }
            if (!ok) break;
            if (PAIR) {
                commit_pair(accf0 + 8 * b);
                commit_pair(mapa(accf0 + 8 * b, 1));
            } else
                mma_commit(accf0 + 8 * b);
        }
    }

    // Warp w holds rows 32 (w % 4) .. + 31 of this CTA's 128, in one half of the columns.
    template <int PHASE, bool SPLIT, class List> __device__ __forceinline__ void store(List &list, int from) {
        constexpr bool SYMMETRIC = symmetric(PHASE);
        static_assert(SYMMETRIC || !SPLIT);
        const int q = warp & 3, half = (warp - 2) >> 2;
        constexpr int UNITS = COLS / 2 / 32;
        // SPLIT: unit `own` of this warp, if any, is this CTA's; `parts` rooms stand behind one another for it, one
        // for each part, the first of them its own
        const int index = 4 * q + 2 * half, own = SPLIT ? ((part - index) & (parts - 1)) : 0;
        uint8_t *const area = smem + STAGES * STAGE_BYTES;
        uint8_t *const rooms = area + (SPLIT ? (index + own) / parts * parts : (warp - 2) * 2) * ROOM;
        const uint32_t rooms_at = smem_u32(rooms), sides0 = sides_at + 16 * (warp - 2);
        const bool failed = PHASE == STEP && __any_sync(0xffffffffu, *(volatile int *)&g_error);
        bool met = false;
        Matrix m;
        Tile tile;
        for (; ok && list.take(m, tile); local++) {
            const Operands p = operands(m, PHASE, from);
            if (failed && m.param) m.rows = 0;  // the epilogue finds no row to update
            const int b = local & 1, ib = tile.i * SIDES + 2 * rank + (q >> 1), r0 = 32 * (q & 1);
            const int hi_to = from ? m.hi[0] : m.hi[1], lo_to_block = from ? m.lo : m.lo2;
            const int jb0 = tile.j * SIDES + half * (SIDES / 2);
            // unit u: columns 32 (u & 1) .. + 31 of block (ib, jb0 + u / 2); all warps' lanes agree on how many there are
            const int units = ib < p.ni ? max(0, min(UNITS, 2 * (p.nj - jb0))) : 0;
            const auto row_of = [&](int u) { return (ib * (SYMMETRIC ? m.sb : m.cb) + jb0 + u / 2) * SIDE + r0; };
            // what the epilogue of a unit reads: A by TMA (a pair where it is fine), or lo of X (where it is fine, F lo was a
            // term), which only this lane reads and writes: straight, the next unit's ahead
            constexpr bool reads = PHASE == QUAD;
            const auto fetch = [&](int u) {
                if (!reads || u >= units) return;
                const uint32_t k = SPLIT ? 0u : (uint32_t)u & 1u;
                pending |= 1u << k;
                if (lane) return;
                const int x = 32 * (u & 1), y = row_of(u);
                mbar_expect_tx(sides0 + 8 * k, m.fine ? ROOM : ROOM / 2);
                if (m.fine) tma_load_2d(rooms_at + k * ROOM + ROOM / 2, &map_units, sides0 + 8 * k, x, (m.gram + m.sb * m.sb) * SIDE + y);
                tma_load_2d(rooms_at + k * ROOM, &map_units, sides0 + 8 * k, x, m.gram * SIDE + y);
            };
            const bool adds = !SYMMETRIC && !m.fine;
            const auto lo_of = [&](int u) {
                return reinterpret_cast<uint4 *>(o.work + (int64_t)(m.lo + ib * m.cb + jb0 + u / 2) * BLOCK_BYTES + lo_at(r0 + lane, 32 * (u & 1)));
            };
            uint4 ahead[4];
            const auto ask = [&](int u) {
                if (!adds || u >= units) return;
                const uint4 *const at = lo_of(u);
#pragma unroll
                for (int e = 0; e < 4; e++) ahead[e] = __ldcg(at + 32 * e);
            };
            if (lane == 0) bulk_wait_read();
            __syncwarp();  // the rooms are free
            ask(0);
            if (SPLIT) {
                fetch(own);
            } else {
                fetch(0);
                fetch(1);
            }
            if (PHASE == STEP && m.param) {  // the parameters are read after the products: into L2 meanwhile, a row a lane
                const int i = ib * SIDE + r0 + lane, j0 = jb0 * SIDE;
#pragma unroll
                for (int j = 0; j < COLS / 2; j += 32)
                    if (i < m.rows && j0 + j < m.cols) asm volatile("prefetch.global.L2 [%0];" ::"l"(m.param + (int64_t)i * m.cols + j0 + j));
            }
            if (!mbar_wait(accf0 + 8 * b, (uint32_t)(local >> 1) & 1u, WAIT_LIMIT)) {
                fail(o, 4);
                ok = false;
                break;
            }
            tc_fence_after();
            if (SPLIT) {
                // the others' units go to their owners
                for (int u = 0; u < units; u++) {
                    if (u == own || part_of(p, SPLIT ? part : 0, SPLIT ? parts : 1) == part_of(p, SPLIT ? part + 1 : 1, SPLIT ? parts : 1)) continue;
                    uint32_t v[32];
                    D1X_TMEM_LD32(tmem + (uint32_t)(b * COLS + half * (COLS / 2) + 32 * u) + ((uint32_t)(32 * q) << 16), v);
                    tmem_wait_ld();
                    const int to = (index + u) & (parts - 1), slot = (index + u) / parts * parts + 1 + (part < to ? part : part - 1);
                    const uint32_t at = mapa(smem_u32(area + slot * ROOM) + lane * 16, to);
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + e * 512), "r"(v[4 * e]), "r"(v[4 * e + 1]),
                                     "r"(v[4 * e + 2]), "r"(v[4 * e + 3])
                                     : "memory");
                }
                __syncwarp();
                cluster_meet();
                met = true;
            }
#pragma unroll 1
            for (int u = SPLIT ? own : 0; u < (SPLIT ? min(units, own + 1) : units); u++) {
                float params[32];
                if (PHASE == STEP && m.param) load_params(m, ib * SIDE + r0, jb0 * SIDE + 32 * u, params);
                uint32_t v[32];
                D1X_TMEM_LD32(tmem + (uint32_t)(b * COLS + half * (COLS / 2) + 32 * u) + ((uint32_t)(32 * q) << 16), v);
                tmem_wait_ld();
                if (SPLIT) {  // a part without a block has left nothing
                    float sum[32] = {};
                    for (int r = 0; r < parts; r++) {
                        if (part_of(p, r, parts) == part_of(p, r + 1, parts)) continue;
                        if (r == part) {
#pragma unroll
                            for (int i = 0; i < 32; i++) sum[i] += __uint_as_float(v[i]);
                            continue;
                        }
                        const float4 *const from = reinterpret_cast<const float4 *>(rooms + (1 + (r < part ? r : r - 1)) * ROOM) + lane;
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            const float4 f = from[32 * e];
                            sum[4 * e] += f.x, sum[4 * e + 1] += f.y, sum[4 * e + 2] += f.z, sum[4 * e + 3] += f.w;
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 32; i++) v[i] = __float_as_uint(sum[i]);
                }
                const uint32_t k = SPLIT ? 0u : (uint32_t)u & 1u;
                if (reads) {
                    pending &= ~(1u << k);
                    turns ^= 1u << k;
                    if (!mbar_wait(sides0 + 8 * k, (turns >> k & 1u) ^ 1u, WAIT_LIMIT)) {
                        fail(o, 5);
                        ok = false;
                        break;
                    }
                } else if (m.fine && u > 1) {  // the room's last contents have been taken away
                    if (lane == 0) bulk_wait_read_but_one();
                    __syncwarp();
                }
                // half a room where that is enough: each of a tile's units has its own
                const uint32_t room_from = SPLIT ? 0u : (PHASE == GRAM || PHASE == APPLY) && !m.fine ? u * (ROOM / 2) : k * ROOM;
                uint8_t *const room = rooms + room_from;
                const uint32_t room_at = rooms_at + room_from;
                const int x0 = 32 * (u & 1), y = row_of(u);
                // this lane's row of 64 bytes: its piece e lies at e ^ (row / 2 & 3), as the TMA's swizzle has it
                uint8_t *const mine = room + lane * 64;
                const auto piece = [&](int e) { return (e ^ (lane >> 1 & 3)) << 4; };
                if constexpr (SYMMETRIC) {
                    const bool diagonal = PHASE == QUAD && ib == jb0 + u / 2 && r0 == x0;  // column i is this lane's own where i == lane
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        float x[8];
                        uint4 hi, lo;
                        if constexpr (PHASE == GRAM) {
#pragma unroll
                            for (int i = 0; i < 8; i++) x[i] = __uint_as_float(v[8 * e + i]) * UNSCALE;
                        } else {
                            float g[8];
                            unpack(*reinterpret_cast<const uint4 *>(mine + piece(e)), g);
#pragma unroll
                            for (int i = 0; i < 8; i++) x[i] = fmaf(NS_C * UNSCALE, __uint_as_float(v[8 * e + i]), NS_B * g[i]);
                            if (m.fine) {
                                unpack(*reinterpret_cast<const uint4 *>(mine + ROOM / 2 + piece(e)), g);
#pragma unroll
                                for (int i = 0; i < 8; i++) x[i] = fmaf(NS_B, g[i], x[i]);
                            }
                            if (diagonal)
#pragma unroll
                                for (int i = 0; i < 8; i++) x[i] += 8 * e + i == lane ? NS_A * SCALE : 0.f;
                        }
                        split(x, hi, lo);
                        *reinterpret_cast<uint4 *>(mine + piece(e)) = hi;
                        if (m.fine) *reinterpret_cast<uint4 *>(mine + ROOM / 2 + piece(e)) = lo;
                    }
                    fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) {
                        const int to = PHASE == GRAM ? m.gram : m.quad;
                        tma_store_2d(&map_units, room_at, x0, to * SIDE + y);
                        if (m.fine) tma_store_2d(&map_units, room_at + ROOM / 2, x0, (to + m.sb * m.sb) * SIDE + y);
                        bulk_commit();
                    }
                } else {
                    float x[32];
                    uint4 *const lo_to = lo_of(u);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
#pragma unroll
                        for (int i = 0; i < 8; i++) x[8 * e + i] = UNSCALE * __uint_as_float(v[8 * e + i]);
                        if (adds) {
                            float l[8];
                            unpack(ahead[e], l);
#pragma unroll
                            for (int i = 0; i < 8; i++) x[8 * e + i] = fmaf(NS_A, l[i], x[8 * e + i]);
                        }
                        if constexpr (PHASE == APPLY) {
                            uint4 hi, lo;
                            split(reinterpret_cast<const float(&)[8]>(x[8 * e]), hi, lo);
                            *reinterpret_cast<uint4 *>(mine + piece(e)) = hi;
                            if (adds)
                                lo_to[32 * e] = lo;
                            else
                                *reinterpret_cast<uint4 *>(mine + ROOM / 2 + piece(e)) = lo;
                        }
                    }
                    if (PHASE == APPLY) ask(u + 1);
                    if constexpr (PHASE == APPLY) {
                        fence_proxy_async();
                        __syncwarp();
                        if (lane == 0) {
                            tma_store_2d(&map_units, room_at, x0, hi_to * SIDE + y);
                            if (m.fine) tma_store_2d(&map_units, room_at + ROOM / 2, x0, lo_to_block * SIDE + y);
                            bulk_commit();
                        }
                    } else {
                        finish(o, m, ib * SIDE + r0, jb0 * SIDE + 32 * u, x, params, reinterpret_cast<float *>(room));
                        ask(u + 1);
                    }
                }
                __syncwarp();
                if (!SPLIT && reads && u + 2 < units) {
                    if (lane == 0) bulk_wait_read();
                    fetch(u + 2);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (PAIR)
                    arrive_cluster(mapa(acce0 + 8 * b, 0));
                else
                    mbar_arrive(acce0 + 8 * b);
            }
        }
        // after an error: loads under way land before the block leaves
        for (uint32_t k = 0; k < 2; k++)
            if (pending >> k & 1u) mbar_wait(sides0 + 8 * k, turns >> k & 1u, WAIT_LIMIT);
        if (lane == 0) bulk_wait();
        if (SPLIT && !met) cluster_meet();
    }
};

// Barriers and tensor memory; the cluster's CTAs have begun when it returns.
template <bool PAIR, bool CLUSTER> __device__ __forceinline__ Roles<PAIR> begin(const CUtensorMap &map, const CUtensorMap &map_units, const Job &o) {
    constexpr int COLS = Roles<PAIR>::COLS;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *const smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *const bars = reinterpret_cast<uint64_t *>(smem + STAGES * STAGE_BYTES + EPI_WARPS * 2 * ROOM), *const sides = bars + 2 * STAGES + 4;
    uint32_t *const tmem_slot = reinterpret_cast<uint32_t *>(sides + 2 * EPI_WARPS);
    const int rank = PAIR ? (int)cluster_rank() : 0, parts = CLUSTER ? (int)cluster_size() : 1, part = CLUSTER ? (int)cluster_rank() : 0;
    Roles<PAIR> r{map, map_units, o, smem, smem_u32(bars), smem_u32(bars + STAGES), smem_u32(bars + 2 * STAGES), smem_u32(bars + 2 * STAGES + 2),
                  smem_u32(sides), 0, (int)threadIdx.x >> 5, (int)threadIdx.x & 31, rank, parts, part};
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; s++) {
            mbar_init(r.full0 + 8 * s, 1);
            mbar_init(r.empty0 + 8 * s, 1);
        }
        for (int b = 0; b < 2; b++) {
            mbar_init(r.accf0 + 8 * b, 1);
            mbar_init(r.acce0 + 8 * b, (PAIR ? 2 : 1) * EPI_WARPS);
        }
        for (int w = 0; w < 2 * EPI_WARPS; w++) mbar_init(r.sides_at + 8 * w, 1);
        mbar_init_fence();
    }
    if (r.warp == 1) {
        if (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(2 * COLS) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(2 * COLS) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    tc_fence_before();
    __syncthreads();
    if (PAIR || CLUSTER) cluster_sync();  // the CTAs' barriers exist before any signal between them
    tc_fence_after();
    r.tmem = *tmem_slot;
    return r;
}
template <bool PAIR> __device__ __forceinline__ void end(const Roles<PAIR> &r) {
    constexpr int COLS = Roles<PAIR>::COLS;
    tc_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync();  // no signal between the CTAs is outstanding past this point
    if (r.warp == 1) {
        tc_fence_after();
        if (PAIR)
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(r.tmem), "r"(2 * COLS) : "memory");
        else
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(r.tmem), "r"(2 * COLS) : "memory");
    }
}

// One product of all matrices by a persistent grid: MODE says what a tile belongs to.
template <int PHASE, int MODE>
__global__ void __launch_bounds__(THREADS, 1) product_kernel(const __grid_constant__ CUtensorMap map, const __grid_constant__ CUtensorMap map_units, const __grid_constant__ Job o) {
    constexpr bool PAIR = MODE == PAIRS, SPLIT = MODE == SPLITS, SYMMETRIC = PHASE == GRAM || PHASE == QUAD;
    pdl_launch();
    Roles<PAIR> roles = begin<PAIR, SPLIT>(map, map_units, o);
    const int together = PAIR ? 2 : roles.parts, first = blockIdx.x / together, step = gridDim.x / together;
    const int tiles = SYMMETRIC ? o.count_symmetric : o.count_full;
    // A plan does not change between the launches of a step (the first of them waits for all that came before), so
    // that a tile is looked up ahead of pdl_wait(), and the next one during the products of this.
    if (!o.matrices) pdl_wait();
    if (roles.warp == 0 && roles.lane == 0) {
        Tiles list(o, SYMMETRIC, tiles, first, step);
        pdl_wait();
        roles.template load<PHASE, SPLIT>(list, o.from);
        roles.loaded();
    } else if (roles.warp == 1 && roles.lane == 0 && roles.rank == 0) {
        Tiles list(o, SYMMETRIC, tiles, first, step);
        pdl_wait();
        roles.template multiply<PHASE, SPLIT>(list, o.from);
    } else if (roles.warp >= 2) {
        Tiles list(o, SYMMETRIC, tiles, first, step);
        pdl_wait();
        roles.template store<PHASE, SPLIT>(list, o.from);
    }
    if (SPLIT && roles.warp < 2) cluster_meet();  // every thread of the cluster comes there once
    end(roles);
}

// All products of small matrices (one tile of A each) in one launch: a cluster takes a matrix through all steps, its CTAs share
// the tiles of X' and, where it is long, the sum of A. A barrier of the cluster stands where the launches' ends stand otherwise:
// 8 x 100 x 800 91 us in place of 111. (What is left are the first loads of each product, a microsecond,
// and instructions: every product's code comes from the far instruction cache each time.)
template <bool DIVIDED>
__global__ void __launch_bounds__(THREADS, 1) small_kernel(const __grid_constant__ CUtensorMap map, const __grid_constant__ CUtensorMap map_units, const __grid_constant__ Job o) {
    Roles<false> roles = begin<false, true>(map, map_units, o);
    const int together = roles.parts, rank = roles.part;
    pdl_wait();
    const Matrix m = matrix_of(o, blockIdx.x / together);
    int from = 0;
    for (int k = 0; k < o.steps; k++, from ^= 1) {
        // a role's share of a product, then the cluster's barrier
        const auto product = [&](auto phase, auto divided, int first, int step) {
            constexpr int PHASE = decltype(phase)::value;
            constexpr bool SPLIT = decltype(divided)::value;
            MatrixTiles list(m, PHASE == GRAM || PHASE == QUAD, first, step);
            if (roles.warp == 0) {
                if (roles.lane == 0) roles.template load<PHASE, SPLIT>(list, from);
            } else if (roles.warp == 1) {
                if (roles.lane == 0) roles.template multiply<PHASE, SPLIT>(list, from);
            } else
                roles.template store<PHASE, SPLIT>(list, from);
            if (SPLIT && roles.warp < 2) cluster_meet();
            // stores by TMA are complete (store() waits for them); loads by TMA come after the barrier, and after what was read
            // of the rooms
            fence_proxy_async();
            cluster_meet();
            if (roles.lane == 0) asm volatile("fence.proxy.async.global;" ::: "memory");
        };
        using One = std::integral_constant<bool, false>;
        if constexpr (DIVIDED)
            product(std::integral_constant<int, GRAM>(), std::integral_constant<bool, true>(), 0, 1);
        else
            product(std::integral_constant<int, GRAM>(), One(), rank, together);
        product(std::integral_constant<int, QUAD>(), One(), rank, together);
        if (k + 1 < o.steps)
            product(std::integral_constant<int, APPLY>(), One(), rank, together);
        else
            product(std::integral_constant<int, STEP>(), One(), rank, together);
    }
    if (roles.warp == 0 && roles.lane == 0) roles.loaded();
    end(roles);
}

#include "muon_narrow.cuh"

// ---------------------------------------------------------------- host side

typedef CUresult (*EncodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                CUtensorMapFloatOOBfill);

// The work buffer's blocks as rows of 64 fp16 elements: whole blocks, and 32 x 32 elements of one.
struct Maps {
    CUtensorMap blocks, units;
};
static int make_maps(Maps &maps, void *work, int64_t blocks) {
    static EncodeTiled encode = nullptr;
    if (!encode) {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q)) return (int)e;
        if (q != cudaDriverEntryPointSuccess) return (int)cudaErrorNotSupported;
        encode = reinterpret_cast<EncodeTiled>(p);
    }
    const cuuint64_t dims[2] = {SIDE, (cuuint64_t)blocks * SIDE}, strides[1] = {128};
    const cuuint32_t one[2] = {1, 1};
    const auto make = [&](CUtensorMap *map, cuuint32_t columns, cuuint32_t rows, CUtensorMapSwizzle swizzle) {
        const cuuint32_t box[2] = {columns, rows};
        return encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, work, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    };
    return make(&maps.blocks, SIDE, SIDE, CU_TENSOR_MAP_SWIZZLE_128B) && make(&maps.units, 32, 32, CU_TENSOR_MAP_SWIZZLE_64B)
               ? 0
               : D1_ERR_BAD_ARGUMENT;
}

typedef void (*Product)(const CUtensorMap, const CUtensorMap, const Job);
static Product product_of(int phase, int mode) {
    static const Product all[3][4] = {
        {product_kernel<GRAM, SINGLES>, product_kernel<QUAD, SINGLES>, product_kernel<APPLY, SINGLES>, product_kernel<STEP, SINGLES>},
        {product_kernel<GRAM, PAIRS>, product_kernel<QUAD, PAIRS>, product_kernel<APPLY, PAIRS>, product_kernel<STEP, PAIRS>},
        {product_kernel<GRAM, SPLITS>, product_kernel<QUAD, SPLITS>, nullptr, nullptr}};  // X' is not divided
    return all[mode][phase];
}
typedef Product Small;
static Small small_of(bool divided) { return divided ? small_kernel<true> : small_kernel<false>; }
static int allow_space() {
    static uint64_t ready = 0;
    int dev = 0;
    if (cudaError_t e = cudaGetDevice(&dev)) return (int)e;
    if (dev < 64 && ((ready >> dev) & 1)) return 0;
    for (int k = 0; k < 12; k++)
        if (const Product p = product_of(k & 3, k >> 2))
            if (cudaError_t e = cudaFuncSetAttribute(p, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES)) return (int)e;
    for (int k = 0; k < 2; k++)
        if (cudaError_t e = cudaFuncSetAttribute(small_of(k), cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES)) return (int)e;
    if (cudaError_t e = cudaFuncSetAttribute(narrow::steps_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, narrow::step_bytes(8))) return (int)e;
    if (cudaError_t e = cudaFuncSetAttribute(narrow::whole_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, narrow::whole_bytes(8))) return (int)e;
    if (dev < 64) ready |= 1ull << dev;
    return 0;
}

static int launch(Job &o, int64_t parts, int64_t blocks, const Load &load, int steps, cudaStream_t s) {
    if (parts > INT32_MAX || load.symmetric > INT32_MAX || load.full > INT32_MAX) return D1_ERR_TOO_LARGE;
    o.count_symmetric = (int)load.symmetric, o.count_full = (int)load.full;
    if (const int e = allow_space()) return e;
    o.steps = steps;
    o.told = told;
    cudaLaunchAttribute attr[2];
    cudaLaunchConfig_t cfg = pdl_config(dim3((unsigned)parts), dim3(PREP), 0, s, attr);
    cfg.numAttrs = 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    if (load.narrow() && steps <= narrow::MOST_STEPS) {
        cudaLaunchConfig_t mid = cfg;
        mid.blockDim = cfg.blockDim = dim3(narrow::THREADS_SUM);
        if (const int n = load.whole_together()) {
            mid.gridDim = dim3((unsigned)(load.matrices * n));
            mid.dynamicSmemBytes = narrow::whole_bytes(load.most_eights);
            mid.attrs = attr + 1, mid.numAttrs = 1;
            attr[1].val.clusterDim.x = n;
            return (int)cudaLaunchKernelEx(&mid, narrow::whole_kernel, o);
        }
        o.adders = (int)std::max<int64_t>(narrow::FEW, 2 * SMS / load.matrices);
        if (cudaError_t e = cudaLaunchKernelEx(&cfg, narrow::sums_kernel, o)) return (int)e;
        const int n = std::min(load.most_parts, o.adders) > narrow::FEW ? load.clusters(8) : 1;
        mid.gridDim = dim3((unsigned)(load.matrices * n));
        mid.dynamicSmemBytes = narrow::step_bytes(load.most_eights);
        mid.numAttrs = 2;
        attr[1].val.clusterDim.x = n;
        if (cudaError_t e = cudaLaunchKernelEx(&mid, narrow::steps_kernel, o)) return (int)e;
        cfg.blockDim = dim3(narrow::THREADS_APPLY);
        cfg.numAttrs = 1;
        return (int)cudaLaunchKernelEx(&cfg, narrow::apply_kernel, o);
    }
    Maps maps;
    if (const int e = make_maps(maps, o.work, blocks)) return e;
    if (cudaError_t e = cudaLaunchKernelEx(&cfg, prepare_kernel<true>, o)) return (int)e;
    cfg.numAttrs = 1;
    if (cudaError_t e = cudaLaunchKernelEx(&cfg, prepare_kernel<false>, o)) return (int)e;
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = SMEM_BYTES;
    if (const int together = load.small_together()) {
        cfg.gridDim = dim3((unsigned)(load.matrices * together));
        cfg.numAttrs = 2;
        attr[1].val.clusterDim.x = together;
        return (int)cudaLaunchKernelEx(&cfg, small_of(together > 1 && saves(load.depth[0], together)), maps.blocks, maps.units, o);
    }
    for (int k = 0; k < steps; k++, o.from ^= 1)
        for (int phase = 0; phase < 3; phase++) {
            const int tiles = phase < 2 ? o.count_symmetric : o.count_full;
            const int split = load.side == 4 || phase == 2 ? 1 : parts_for(tiles, load.depth[phase > 0]);
            const int together = load.side == 4 ? 2 : split, most = SMS / together, n = tiles < most ? tiles : most;
            cfg.gridDim = dim3((unsigned)(n * together));
            cfg.numAttrs = together > 1 ? 2 : 1;
            attr[1].val.clusterDim.x = together;
            const Product kernel = product_of(phase == 2 && k == steps - 1 ? STEP : phase, load.side == 4 ? PAIRS : split > 1 ? SPLITS : SINGLES);
            if (cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, maps.blocks, maps.units, o)) return (int)e;
        }
    return 0;
}

}  // namespace muon
}  // namespace d1

using namespace d1::muon;

// Sizes of a plan, and the plan itself when `out` is not NULL.
static int plan(const D1MuonTensor *tensors, int n, float *momentum, Plan &head, uint8_t *out) {
    if (!tensors || n < 1) return D1_ERR_BAD_ARGUMENT;
    head = Plan{};
    Load small = load_of(2), large = load_of(4);
    int64_t block = 0, part = 0;
    for (int t = 0; t < n; t++) {
        const D1MuonTensor &d = tensors[t];
        const int64_t need = blocks_needed(d.rows, d.cols, d.precise != 0);
        if (need < 0 || d.count < 0 || d.count > MOST_BLOCKS) return D1_ERR_BAD_ARGUMENT;
        if (need * d.count + block > MOST_BLOCKS) return D1_ERR_TOO_LARGE;
        if (!d.count) continue;
        Matrix m;
        int64_t from = block, from_part = part;
        place(m, d.rows, d.cols, from, from_part, d.precise != 0);
        block += (from - block) * d.count, part += (from_part - part) * d.count;
        head.matrices += d.count;
        small.add(m, d.count);
        large.add(m, d.count);
    }
    head.parts = part;
    head.blocks = block;
    head.load = large.microseconds() < small.microseconds() ? large : small;
    if (!head.matrices) return D1_ERR_BAD_ARGUMENT;
    if (head.load.symmetric > INT32_MAX || head.load.full > INT32_MAX || head.parts > INT32_MAX) return D1_ERR_TOO_LARGE;
    head.at_matrices = (sizeof(Plan) + 15) / 16 * 16;
    head.at_parts = head.at_matrices + head.matrices * (int64_t)sizeof(Matrix);
    head.at_symmetric = head.at_parts + head.parts * (int64_t)sizeof(Part);
    head.at_full = head.at_symmetric + head.load.symmetric * (int64_t)sizeof(Tile);
    head.bytes = head.at_full + head.load.full * (int64_t)sizeof(Tile);
    if (!out) return 0;
    *(Plan *)out = head;
    Matrix *const matrices = (Matrix *)(out + head.at_matrices);
    Part *parts = (Part *)(out + head.at_parts);
    int64_t momentum_at = 0;
    int k = 0;
    block = part = 0;
    for (int t = 0; t < n; t++) {
        const D1MuonTensor &d = tensors[t];
        const int64_t size = d.rows * d.cols, grad_size = d.grad_type == D1_TYPE_F32 ? 4 : 2;
        for (int64_t c = 0; c < d.count; c++, k++) {
            Matrix m{};
            place(m, d.rows, d.cols, block, part, d.precise != 0);
            m.param = d.param + c * size;
            m.grad = (const char *)d.grad + c * size * grad_size;
            m.out = d.copy ? (char *)d.copy + c * size * 2 : nullptr;
            m.momentum = momentum + momentum_at + c * size;
            m.pitch = d.cols;
            m.grad_type = d.grad_type;
            m.out_type = D1_TYPE_BF16;
            m.rate = (float)(0.2 * sqrt((double)(d.rows > d.cols ? d.rows : d.cols)));
            m.keep_decay = (float)d.decay;
            matrices[k] = m;
            for (int p = 0; p < m.parts; p++) *parts++ = Part{k, p};
        }
        momentum_at += (size * d.count + 127) / 128 * 128;
    }
    // the longest sums first, so that the last tiles to be taken are short ones
    int *const order = new (std::nothrow) int[head.matrices];
    if (!order) return D1_ERR_TOO_LARGE;
    for (int i = 0; i < k; i++) order[i] = i;
    const auto list = [&](Tile *to, bool symmetric) {
        std::stable_sort(order, order + k, [&](int a, int b) {
            const auto depth = [&](const Matrix &m) { return symmetric ? (m.tall ? m.rb : m.cb) : m.sb; };
            return depth(matrices[a]) > depth(matrices[b]);
        });
        for (int q = 0; q < k; q++) {
            const Matrix &m = matrices[order[q]];
            const int64_t count = symmetric ? symmetric_tiles(m, head.load.side) : full_tiles(m, head.load.side);
            for (int t = 0; t < (int)count; t++) {
                int i, j;
                if (symmetric)
                    symmetric_tile(t, i, j);
                else
                    grouped_tile(t, tiles_of(m.rb, head.load.side), tiles_of(m.cb, head.load.side), i, j);
                *to++ = Tile{order[q], (uint16_t)i, (uint16_t)j};
            }
        }
    };
    list((Tile *)(out + head.at_symmetric), true);
    list((Tile *)(out + head.at_full), false);
    delete[] order;
    return 0;
}

static int64_t bytes_of(int64_t blocks, int64_t parts) { return work_blocks_bytes(blocks) + parts * 8; }

extern "C" int64_t d1_muon_plan_bytes(const D1MuonTensor *tensors, int ntensors) {
    Plan head;
    return plan(tensors, ntensors, nullptr, head, nullptr) ? -1 : head.bytes;
}
extern "C" int64_t d1_muon_work_bytes(const D1MuonTensor *tensors, int ntensors) {
    Plan head;
    return plan(tensors, ntensors, nullptr, head, nullptr) ? -1 : bytes_of(head.blocks, head.parts);
}

extern "C" int d1_muon_plan(const D1MuonTensor *tensors, int ntensors, float *momentum, void *host_plan, int64_t bytes) {
    Plan head;
    if (const int e = plan(tensors, ntensors, momentum, head, nullptr)) return e;
    if (!momentum || !host_plan || bytes < head.bytes || !d1::aligned_to(8, host_plan) || !d1::aligned_to(16, momentum)) return D1_ERR_BAD_ARGUMENT;
    for (int i = 0; i < ntensors; i++) {
        const D1MuonTensor &t = tensors[i];
        if (t.count && (!t.param || !t.grad || (t.grad_type != D1_TYPE_F32 && t.grad_type != D1_TYPE_BF16) || !(t.decay == t.decay) ||
                        !d1::aligned_to(4, t.param) || !d1::element_aligned(t.grad, t.grad_type) || !d1::aligned_to(2, t.copy)))
            return D1_ERR_BAD_ARGUMENT;
    }
    return plan(tensors, ntensors, momentum, head, (uint8_t *)host_plan);
}

extern "C" int d1_muon(const void *host_plan, const void *device_plan, double lr, double momentum, int nesterov, int steps, void *work,
                       void *stream) {
    if (!host_plan || !device_plan || !work || steps < 1 || steps > 64 || !(momentum >= 0. && momentum < 1.) || !(lr == lr) ||
        !d1::aligned_to(8, host_plan, device_plan) || !d1::aligned_to(128, work))
        return D1_ERR_BAD_ARGUMENT;
    const Plan &head = *(const Plan *)host_plan;
    const uint8_t *const at = (const uint8_t *)device_plan;
    Job o{};
    o.matrices = (const Matrix *)(at + head.at_matrices);
    o.parts = (const Part *)(at + head.at_parts);
    o.symmetric = (const Tile *)(at + head.at_symmetric);
    o.full = (const Tile *)(at + head.at_full);
    o.work = (uint8_t *)work;
    o.partials = (double *)(o.work + work_blocks_bytes(head.blocks));
    o.mu = (float)momentum, o.nesterov = nesterov != 0, o.lr = lr;
    return launch(o, head.parts, head.blocks, head.load, steps, (cudaStream_t)stream);
}

// The stack's one matrix, its blocks and parts; false when it is out of range.
static bool stack(int64_t count, int64_t rows, int64_t cols, bool precise, Matrix &m, int64_t &blocks, int64_t &parts) {
    const int64_t need = blocks_needed(rows, cols, precise);
    if (need < 0 || count < 0 || count > MOST_BLOCKS || need * count > MOST_BLOCKS) return false;
    m = Matrix{};
    blocks = parts = 0;
    place(m, rows, cols, blocks, parts, precise);
    return true;
}

static int64_t stack_bytes(int64_t count, int64_t rows, int64_t cols, bool precise) {
    Matrix m;
    int64_t blocks, parts;
    return stack(count, rows, cols, precise, m, blocks, parts) ? bytes_of(count * blocks, count * parts) : -1;
}

static int orthogonalize(const void *x, int64_t ldx, int64_t x_step, int type, int64_t count, int64_t rows, int64_t cols, void *y, int y_type, int steps,
                         bool precise, void *work, void *stream) {
    Matrix m;
    int64_t blocks, parts;
    if (!d1::type_ok(type) || (y_type != D1_TYPE_BF16 && y_type != D1_TYPE_F16) || !stack(count, rows, cols, precise, m, blocks, parts) || steps < 1 ||
        steps > 64 || (count && (!x || !y || !work)) || ldx < 0 || x_step < 0 || ldx > ((int64_t)1 << 42) || x_step > ((int64_t)1 << 42) ||
        !d1::element_aligned(x, type) || !d1::aligned_to(2, y) || !d1::aligned_to(128, work))
        return D1_ERR_BAD_ARGUMENT;
    if (count == 0) return 0;
    const int64_t size = type == D1_TYPE_F32 ? 4 : 2;
    // the result shares no memory with the range of x
    const uintptr_t a = (uintptr_t)x, b = (uintptr_t)y;
    if (a < b + (uintptr_t)(count * rows * cols * 2) && b < a + (uintptr_t)(((count - 1) * x_step + (rows - 1) * ldx + cols) * size))
        return D1_ERR_BAD_ARGUMENT;
    m.grad = x, m.grad_type = type, m.pitch = ldx;
    m.out = y, m.out_type = y_type;
    Job o{};
    o.one = m;
    o.grad_step = x_step * size, o.out_step = rows * cols * 2;
    o.block_step = (int)blocks;
    Load small = load_of(2), large = load_of(4);
    small.add(m, count);
    large.add(m, count);
    const Load &load = large.microseconds() < small.microseconds() ? large : small;
    if (load.symmetric > INT32_MAX || load.full > INT32_MAX) return D1_ERR_TOO_LARGE;
    o.per_symmetric = (int)(load.symmetric / count), o.per_full = (int)(load.full / count);
    o.tm = tiles_of(m.rb, load.side), o.tn = tiles_of(m.cb, load.side);
    o.work = (uint8_t *)work;
    o.partials = (double *)(o.work + work_blocks_bytes(count * blocks));
    return launch(o, count * parts, count * blocks, load, steps, (cudaStream_t)stream);
}

extern "C" int64_t d1_orthogonalize_work_bytes(int64_t count, int64_t rows, int64_t cols) { return stack_bytes(count, rows, cols, false); }
extern "C" int d1_orthogonalize(const void *x, int64_t ldx, int64_t x_step, int type, int64_t count, int64_t rows, int64_t cols, void *y, int y_type,
                                int steps, void *work, void *stream) {
    return orthogonalize(x, ldx, x_step, type, count, rows, cols, y, y_type, steps, false, work, stream);
}
extern "C" int64_t d1_orthogonalize_precise_work_bytes(int64_t count, int64_t rows, int64_t cols) { return stack_bytes(count, rows, cols, true); }
extern "C" int d1_orthogonalize_precise(const void *x, int64_t ldx, int64_t x_step, int type, int64_t count, int64_t rows, int64_t cols, void *y,
                                        int y_type, int steps, void *work, void *stream) {
    return orthogonalize(x, ldx, x_step, type, count, rows, cols, y, y_type, steps, true, work, stream);
}

// Last error recorded by a wait that ran out (0 = none); clears it.
extern "C" int d1_muon_error(void) {
    int h = 0, z = 0;
    if (cudaMemcpyFromSymbol(&h, g_error, sizeof(int)) != cudaSuccess) return -1;
    if (h) cudaMemcpyToSymbol(g_error, &z, sizeof(int));
    if (int *const p = told) *p = 0;
    return h;
}
extern "C" int d1_muon_error_flag(int *flag) {
    if (!d1::aligned_to(4, flag)) return D1_ERR_BAD_ARGUMENT;
    told = flag;
    return 0;
}
extern "C" int d1_muon_set_error(int code) {
    if (cudaError_t e = cudaMemcpyToSymbol(g_error, &code, sizeof(int))) return (int)e;
    if (int *const p = told) *p = code;
    return 0;
}
