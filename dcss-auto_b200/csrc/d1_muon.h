// How the Newton-Schulz products lay out and divide their work, by plain
// arithmetic (no CUDA type or call, so that it is checked on the host).
//
// All 16-bit operands live in one buffer of blocks: 64 x 64 elements in 64 rows
// of 128 bytes, so that one tensor map of 64-element rows serves every matrix
// and a block is an operand of the tensor cores in either orientation. A matrix
// of r x c elements has ceil(r / 64) x ceil(c / 64) blocks, row of blocks after
// row of blocks, zero past its edges; products of zeros keep them zero.
#pragma once
#include <math.h>
#include <stdint.h>

#include "../../include/d1.h"

#ifdef __CUDACC__
#define D1_MUON_BOTH __host__ __device__ __forceinline__
#else
#define D1_MUON_BOTH inline
#endif

namespace d1 {
namespace muon {

constexpr int SIDE = 64, BLOCK_BYTES = SIDE * SIDE * 2;
constexpr int MOST_PARTS = 256;  // partial sums of one matrix's norm
constexpr int64_t MOST_BLOCKS = (int64_t)1 << 24;  // rows of the tensor map stay below 2^30

// One matrix. X is held as hi + lo, hi twice (a product reads one and writes the other).
struct Matrix {
    float *param;         // Muon: the master (NULL: orthogonalize)
    const void *grad;     // the gradient, or the matrix to orthogonalize
    void *out;            // Muon: the bf16 copy or NULL; orthogonalize: the result
    float *momentum;      // Muon
    int64_t pitch;        // elements between rows of grad (param, out and momentum are contiguous)
    int rows, cols;       // of the matrix
    int rb, cb;           // of its blocks
    int sb;               // blocks along the smaller side
    int tall;             // rows > cols: the Gram matrix is X^T X
    int hi[2], lo, gram, quad;  // first blocks
    int lo2;              // where a product writes lo when it reads the first one; the same where each tile reads its own only
    int fine;             // A and F are pairs too (lo sb * sb blocks after hi), and products take all three terms
    int part0, parts;     // partial sums of the norm
    int grad_type, out_type;
    float rate, keep_decay;  // 0.2 sqrt(max(rows, cols)); the weight decay
};

// A tile of a product: row and column of tiles.
struct Tile {
    int matrix;
    uint16_t i, j;
};
// The blocks k, k + parts, ... of a matrix, k < parts.
struct Part {
    int matrix, k;
};

D1_MUON_BOTH int blocks_of(int64_t n) { return (int)((n + SIDE - 1) / SIDE); }
D1_MUON_BOTH int tiles_of(int blocks, int side) { return (blocks + side - 1) / side; }

// Whether all products take three terms: where the caller asks for it, and with one block along the smaller side.
D1_MUON_BOTH bool is_fine(int64_t sb, bool precise) { return precise || sb == 1; }
// Blocks of A, or of F: a pair where it is fine.
D1_MUON_BOTH int64_t gram_blocks(int64_t sb, bool precise) { return is_fine(sb, precise) ? 2 * sb * sb : sb * sb; }
// Blocks of X: hi twice and lo, which a product of pairs may read and write in one place where a tile has all of the sum.
D1_MUON_BOTH int64_t x_blocks(int64_t n, int64_t sb, bool precise) { return precise && sb > 1 ? 4 * n : 3 * n; }

// Sizes, blocks (from `block` on) and parts (from `part` on) of a matrix; moves both on.
inline void place(Matrix &m, int64_t rows, int64_t cols, int64_t &block, int64_t &part, bool precise = false) {
    m.rows = (int)rows, m.cols = (int)cols;
    m.rb = blocks_of(rows), m.cb = blocks_of(cols);
    m.tall = rows > cols;
    m.sb = m.tall ? m.cb : m.rb;
    m.fine = is_fine(m.sb, precise);
    const int64_t n = (int64_t)m.rb * m.cb, s = gram_blocks(m.sb, precise), x = x_blocks(n, m.sb, precise);
    m.hi[0] = (int)block;
    m.hi[1] = (int)(block + n);
    m.lo = (int)(block + 2 * n);
    m.lo2 = x > 3 * n ? (int)(block + 3 * n) : m.lo;
    m.gram = (int)(block + x);
    m.quad = (int)(block + x + s);
    block += x + 2 * s;
    m.part0 = (int)part;
    m.parts = (int)(n < MOST_PARTS ? n : MOST_PARTS);
    part += m.parts;
}
// Blocks that place() takes; -1 for a matrix that is out of range.
inline int64_t blocks_needed(int64_t rows, int64_t cols, bool precise = false) {
    if (rows < 1 || cols < 1 || rows > ((int64_t)1 << 21) || cols > ((int64_t)1 << 21)) return -1;
    const int64_t rb = blocks_of(rows), cb = blocks_of(cols), sb = rows > cols ? cb : rb;
    return x_blocks(rb * cb, sb, precise) + 2 * gram_blocks(sb, precise);
}

// Tile t of a symmetric matrix of tiles: row i >= column j, row after row. (In 32 bits and from a root, because the kernels
// do it for every tile: t < 2^31.)
D1_MUON_BOTH void symmetric_tile(int t, int &i, int &j) {
    int r = (int)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);  // off by a little where t has more than 24 bits
    while ((int64_t)r * (r + 1) / 2 > t) r--;
    while ((int64_t)(r + 1) * (r + 2) / 2 <= t) r++;
    i = r;
    j = (int)(t - (int64_t)r * (r + 1) / 2);
}
// Tile t of tm x tn: eight rows of tiles at a time, column after column, so that tiles that
// run together share operands in L2.
D1_MUON_BOTH void grouped_tile(int t, int tm, int tn, int &i, int &j) {
    const int per = 8 * tn, g = t / per, r = t - g * per;
    const int high = tm - 8 * g < 8 ? tm - 8 * g : 8;
    i = 8 * g + r % high;
    j = r / high;
}

D1_MUON_BOTH int64_t symmetric_tiles(const Matrix &m, int side) {
    const int64_t n = tiles_of(m.sb, side);
    return n * (n + 1) / 2;
}
D1_MUON_BOTH int64_t full_tiles(const Matrix &m, int side) { return (int64_t)tiles_of(m.rb, side) * tiles_of(m.cb, side); }

// CTAs that share the sum of `depth` blocks of each of a few tiles: as many as there is room for, while it saves ten
// blocks' time (the exchange of the parts costs some five).
inline int room(int n) { return n == 8 ? 112 : n == 4 ? 128 : 148; }  // what clusters of n CTAs find room for at once
inline bool saves(int depth, int parts) { return depth - depth / parts >= 10; }
inline int parts_for(int64_t tiles, int depth) {
    int parts = 1;
    for (int n = 2; n <= 8; n *= 2)
        if (tiles * n <= room(n) && saves(depth, n)) parts = n;
    return parts;
}

// What a step is made of with tiles of `side` blocks, and about how long it takes.
struct Load {
    int side;
    int64_t symmetric, full;  // tiles
    int depth[2];             // the longest sums, in blocks, of A and of the other products
    double work[3];           // blocks of all sums, by product
    int64_t matrices;
    int widest, longest;      // the most tiles along a smaller side, and of one X'
    int64_t wider;            // matrices whose smaller side has more than one block
    int most_parts, most_eights;  // of one matrix; of a smaller side, in eights

    void add(const Matrix &m, int64_t count) {
        const int64_t s = symmetric_tiles(m, side) * count, f = full_tiles(m, side) * count;
        const int terms = m.fine ? 3 : 1, first = (m.tall ? m.rb : m.cb) * terms, others = m.sb * terms;
        const int wide = tiles_of(m.sb, side), most = (int)full_tiles(m, side);
        matrices += count;
        if (m.sb > 1) wider += count;
        if (m.parts > most_parts) most_parts = m.parts;
        const int eights = ((m.tall ? m.cols : m.rows) + 7) / 8;
        if (eights > most_eights) most_eights = eights;
        if (wide > widest) widest = wide;
        if (most > longest) longest = most;
        symmetric += s, full += f;
        work[0] += (double)s * first, work[1] += (double)s * others, work[2] += (double)f * others;
        if (first > depth[0]) depth[0] = first;
        if (others > depth[1]) depth[1] = others;
    }
    // Whether the steps are taken without X (muon_narrow.cuh). Beside other matrices the narrow ones go with those through
    // their launches at no cost (the conv policy's six take 140 us in one graph, its two wide ones 141 without the four narrow ones).
    bool narrow() const { return wider == 0; }
    // Blocks of a cluster for each matrix, n at most, so that all clusters run at once.
    int clusters(int n) const {
        while (n > 1 && matrices * n > room(n)) n /= 2;
        return n;
    }
    // Blocks of the cluster that takes a narrow matrix through everything in one launch, 0 where that is not done: a block has two
    // of its blocks of X at most, one in the largest clusters of wider ones (three launches and one: 8 x 1,000 13.5 and 12.6 us,
    // 100 x 60 x 120 55 and 48, but 48 x 1,000 30.7 and 32.0, 64 x 1,000 46 and 52).
    int whole_together() const {
        int n = 1;
        while (n < 8 && n < most_parts) n *= 2;
        n = clusters(n);
        return most_parts <= (n == 8 && most_eights > 4 ? n : 2 * n) ? n : 0;
    }
    // CTAs of the cluster that takes each matrix through all products in one launch, 0 where that is not done: every
    // matrix has one tile of A and no more than two of X' a CTA (128 x 4,000, with four, took 138 us in place of the launches'
    // 121), and all clusters run at once.
    int small_together() const {
        if (side != 2 || widest > 1) return 0;
        int n = 1;
        while (n < 8 && (n < longest || (!saves(depth[0], n) && saves(depth[0], 2 * n)))) n *= 2;
        n = clusters(n);
        return matrices * n <= 148 && longest <= 2 * n ? n : 0;
    }
    // A block of 64 of the sum takes a pair of CTAs 0.43 us for a tile of 256 x 256, a CTA 0.5 us for one of 128 x 128 (both measured with the
    // GPU full: the one is bound by shared memory, the other by what comes from L2); a pair's launches take 8 us more in all.
    double microseconds() const {
        double sum = side == 4 ? 8. : 0.;
        for (int k = 0; k < 3; k++) {
            const int parts = side == 4 || k == 2 ? 1 : parts_for(symmetric, depth[k > 0]);
            const double even = work[k] / (side == 4 ? 74 : 148), longest = (double)depth[k > 0] / parts;
            sum += (side == 4 ? 0.43 : 0.5) * (even > longest ? even : longest);
        }
        return sum;
    }
};
inline Load load_of(int side) { return Load{side, 0, 0, {0, 0}, {0., 0., 0.}, 0, 0, 0, 0, 0, 0}; }

// What a plan begins with: sizes of its lists and where they start (bytes).
struct Plan {
    int64_t bytes, matrices, parts;
    int64_t at_matrices, at_parts, at_symmetric, at_full;
    int64_t blocks;  // of the work buffer
    Load load;
};

D1_MUON_BOTH int64_t work_blocks_bytes(int64_t blocks) { return blocks * BLOCK_BYTES; }

}  // namespace muon
}  // namespace d1
