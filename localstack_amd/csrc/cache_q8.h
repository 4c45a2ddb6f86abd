// cache_q8.h - the record of a page of 32 cells and a KV head in a quantised cache.
//
// A value of 32 dims of a cell is d q: d is the smallest fp16 number that is no less than their largest magnitude over 127, q the
// whole number in [-127, 127] nearest to value / d (halves to the even one). A record is 68 HD bytes, one after the other: K's q,
// K's d, V's q, V's d. The q lie as the matrix products of attention take them, 16 bytes a lane (lane = 16 a + r, 64 lanes):
//   K: [m = HD / 32][lane][2 tiles][8 dims]  row r of tile t is cell 8 (r / 4) + 4 t + r % 4; dims 32 m + 8 a + 0 .. 7
//   V: [m = HD / 32][lane][2 tiles][8 cells] row r of tile t is dim 32 m + 16 t + r; cells 8 a + 0 .. 7
//   d: [m = HD / 32][32 cells]
// so a lane's load is an operand of two 16 x 16 x 32 products, a wavefront's load is 1 KiB in a row, and the results of the first
// product leave a lane with cells 8 a + 0 .. 7 of one query head, which is what the second one takes. Blocks of 32 dims with a
// scale each are Q8_0's (8.5 bits a value); a scale for a whole row of 128 would save 4% of the bytes, and lose what the other
// dims hold wherever one dim is large.
#pragma once

#include "batch.h"

namespace lstk {

constexpr int kQ8Dims = 32; // of a scale

__host__ __device__ constexpr int q8_record(int hd) { return 68 * hd; }
__host__ __device__ constexpr int q8_k(int m, int cell, int d) { // d: in [0, 32)
    return m * 1024 + (d / 8 * 16 + cell / 8 * 4 + cell % 4) * 16 + cell / 4 % 2 * 8 + d % 8;
}
__host__ __device__ constexpr int q8_v(int hd, int m, int cell, int d) {
    return 34 * hd + m * 1024 + (cell / 8 * 16 + d % 16) * 16 + d / 16 * 8 + cell % 8;
}
__host__ __device__ constexpr int q8_k_scale(int hd, int m, int cell) { return 32 * hd + (m * 32 + cell) * 2; }
__host__ __device__ constexpr int q8_v_scale(int hd, int m, int cell) { return 66 * hd + (m * 32 + cell) * 2; }

}  // namespace lstk
