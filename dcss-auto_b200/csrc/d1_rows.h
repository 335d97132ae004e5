// Where the rows of a matrix lie in memory, by plain arithmetic on addresses
// (no CUDA type or call, so that it is checked on the host).
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define D1_ROWS_BOTH __host__ __device__ __forceinline__
#else
#define D1_ROWS_BOTH inline
#endif

namespace d1 {

// `count` rows of `width` bytes, `pitch` bytes apart.
struct RowSpan {
    uintptr_t at;
    int64_t count, width, pitch;
};

// Whether two such sets of rows share a byte. Exact: the rows of one may lie
// between those of the other, as two column slices of one buffer do.
inline bool rows_overlap(RowSpan a, RowSpan b) {
    if (a.count < 1 || b.count < 1 || a.width < 1 || b.width < 1) return false;
    if (a.pitch == 0) a.count = 1;  // one row, again and again
    if (b.pitch == 0) b.count = 1;
    const uintptr_t a_end = a.at + (uintptr_t)((a.count - 1) * a.pitch + a.width), b_end = b.at + (uintptr_t)((b.count - 1) * b.pitch + b.width);
    if (a.at >= b_end || b.at >= a_end) return false;
    if (a.count == 1) a.pitch = b.pitch;
    if (b.count == 1) b.pitch = a.pitch;
    if (a.count == 1 && b.count == 1) return true;
    if (a.pitch != b.pitch) {  // row by row of the one that has fewer
        const bool first = a.count <= b.count;
        RowSpan one = first ? a : b;
        const RowSpan other = first ? b : a;
        const int64_t n = one.count, step = one.pitch;
        one.count = 1;
        for (int64_t i = 0; i < n; i++, one.at += (uintptr_t)step)
            if (rows_overlap(one, other)) return true;
        return false;
    }
    // rows i of a and j of b meet where d - a.width < k pitch < d + b.width with k = i - j
    const int64_t d = (int64_t)(b.at - a.at), low = d - a.width, p = a.pitch;
    int64_t k = (low >= 0 ? low / p : -((-low + p - 1) / p)) + 1;
    if (k < 1 - b.count) k = 1 - b.count;
    return k < a.count && k * p < d + b.width;
}

// The 16-byte piece at offset p (a multiple of 16) of a row of `size` bytes,
// counted from the last 16-byte boundary at or before it: where it is copied from and
// how many of its bytes are read. A piece past the row's end reads nothing, but a
// copy's source is aligned whatever its size, so there it is that boundary.
struct RowPiece {
    uintptr_t from;
    int bytes;
};
D1_ROWS_BOTH RowPiece row_piece(uintptr_t row, int size, int p) {
    const uintptr_t base = row & ~(uintptr_t)15;
    const int left = (int)(row & 15) + size - p;
    return {left > 0 ? base + p : base, left < 0 ? 0 : left < 16 ? left : 16};
}

}  // namespace d1
