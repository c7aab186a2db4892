// Tiles of input rows of a product, whole or by expert, and the rows behind them.
#pragma once

#include "mx4.h"

namespace spa {
namespace mx {

struct Tile {
    int expert, first, rows;             // of the rows (whole), or of the slots in their experts' order
};

// The tiles that there may be: every expert with rows has one that is not full.
inline int64_t most_tiles(const Product& p, int height) {
    if (!p.experts) return ((int64_t)p.m + height - 1) / height;
    return p.m / height + (p.m < p.experts ? p.m : p.experts);
}

// a lane's expert e: its first slot and the end, which lie in 0..m whatever the numbers are
struct Span { int begin, end; };
__device__ __forceinline__ Span span_of(const Product& p, int e) {
    if (e >= p.experts) return Span{0, 0};
    const int begin = tmin(tmax(p.starts[e], 0), p.m);
    return Span{begin, tmin(tmax(p.starts[e + 1], begin), p.m)};
}

// the tiles that there are
__device__ __forceinline__ int tiles_of(const Product& p, int height) {
    int sum = 0;
    for (int e = threadIdx.x & 63; e < p.experts; e += 64) {
        const Span s = span_of(p, e);
        sum += (s.end - s.begin + height - 1) / height;
    }
#pragma unroll
    for (int s = 32; s; s >>= 1) sum += __shfl_xor(sum, s);
    return __builtin_amdgcn_readfirstlane(sum);
}

// Tile `id` of `height` rows; no rows behind the last. An expert's tiles follow those of the experts before it: each
// lane counts the tiles of its own, 64 experts at a time.
__device__ __forceinline__ Tile tile_at(const Product& p, int id, int height) {
    if (!p.experts) {
        const int first = id * height;
        return Tile{0, first, first < p.m ? tmin(height, p.m - first) : 0};
    }
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int e0 = 0; e0 < p.experts; e0 += 64) {
        const auto [begin, end] = span_of(p, e0 + lane);
        const int own = (end - begin + height - 1) / height;
        int sum = own;
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) {
            const int v = __shfl_up(sum, s);
            if (lane >= s) sum += v;
        }
        const uint64_t past = __ballot(before + sum > id);
        if (past) {
            const int at = __builtin_ctzll(past);
            const int b = __shfl(begin, at), n = __shfl(end, at), in = id - before - __shfl(sum - own, at);
            const int first = b + in * height;
            return Tile{__builtin_amdgcn_readfirstlane(e0 + at), __builtin_amdgcn_readfirstlane(first),
                        __builtin_amdgcn_readfirstlane(tmin(height, n - first))};
        }
        before += __shfl(sum, 63);
    }
    return Tile{0, 0, 0};
}

// What a tile's row `at` is: the output's row, -1 of a slot outside 0..m-1, which has none; and the input's (the first, of such
// a slot)
__device__ __forceinline__ int output_row(const Product& p, int at) {
    if (!p.experts) return at;
    const int slot = p.order[at];
    return (uint32_t)slot < (uint32_t)p.m ? slot : -1;
}
__device__ __forceinline__ int input_row(const Product& p, int output) { return p.experts ? tmax(output, 0) / p.each : output; }

}  // namespace mx
}  // namespace spa
