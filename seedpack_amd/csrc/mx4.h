// 4-bit floating point in microscaled blocks: what its kernels share (mx4.hip, mx4_product.hip).
//
// A matrix is codes, 16 bytes for each block of 32 numbers along a row, and scales, a byte a block. Number j of a block is
// in the low half of byte j, number j + 16 in the high half of it, as GGUF's MXFP4 blocks hold them behind their
// scale's byte. A code is a sign, two bits of exponent and one of mantissa (0 .5 1 1.5 2 3 4 6), a scale b stands for
// 2^(b - 127), 255 for a block of NaN. Each row has `pitch` blocks, a multiple of 8 (128 bytes of codes, the step
// of the products): those behind its numbers are zeros.
#pragma once

#include "linear.h"

namespace spa {
namespace mx {

inline int64_t pitch_of(int64_t cols) { return (cols + 255) / 256 * 8; }

// the operands and results of a product, whole or by expert
struct Product {
    const uint8_t *xc, *xs;              // m rows of inputs, or with order the rows that the slots name
    const uint8_t *w0c, *w0s, *w1c, *w1s;
    int pitch;                           // blocks of a row
    int m, n;                            // rows or slots; outputs
    int experts;                         // 0: one matrix for all rows
    const int32_t *order, *starts;
    int each;                            // slot p takes row p / each
    uint32_t magic;                      // the upper half of p times it is p / each; 0: divide
    void* y;
    int64_t ldy;
    int kind, act;
    int pieces;                          // of k, whose float32 sums are joined by a second launch; 1: none
    float* part;                         // [pieces, of the gate's and of the up projection][m][n]
};

// A workgroup's waves of a product of few rows, and how many of them share their rows: as many as there are pieces of 512 of k
constexpr int FEW_WAVES = 8;
inline int few_split(int pitch) {
    int split = 1;
    while (split < FEW_WAVES && 2 * split <= (pitch + 15) / 16) split *= 2;
    return split;
}

int product_few(const Product& p, bool wide, hipStream_t st);   // wide: 32 x 32 outputs a wave, of one matrix
int product_many(const Product& p, bool large, hipStream_t st);

}  // namespace mx
}  // namespace spa
