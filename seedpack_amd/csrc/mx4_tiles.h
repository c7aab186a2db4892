// Tiles of input rows of a product, whole or by expert, and the rows behind them.
#pragma once

#include "mx4.h"

namespace spa {
namespace mx {

struct Tile {
    int expert, first, rows;             // of the rows (whole), or of the slots in their experts' order
};

// The tiles that there may be: every expert with rows has one that is not full.
__host__ __device__ inline int most_tiles(const Product& p, int height) {
    if (!p.experts) return (p.m + height - 1) / height;
    return p.m / height + (p.m < p.experts ? p.m : p.experts);
}

// a lane's expert e: its first slot and the end, which lie in 0..m whatever the numbers are
struct Span { int begin, end; };
__device__ __forceinline__ Span span_of(const Product& p, int e) {
    if (e >= p.experts) return Span{0, 0};
    const int begin = tmin(tmax(p.starts[e], 0), p.m);
    return Span{begin, tmin(tmax(p.starts[e + 1], begin), p.m)};
}

// inclusive sums over the wave
__device__ __forceinline__ int running(int v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const int t = __shfl_up(v, s);
        if (lane >= s) v += t;
    }
    return v;
}

// The tiles of a product of up to 64 experts, an expert a lane; of more experts they are counted again for each question.
struct Tiles {
    Span span;
    int own, sum, total;                 // an expert's tiles, with those before it, and all
};
__device__ __forceinline__ Tiles tiles_of(const Product& p, int height) {
    const int lane = threadIdx.x & 63;
    Tiles t{};
    if (!p.experts) {
        t.total = (p.m + height - 1) / height;
        return t;
    }
    for (int e0 = 0; e0 < p.experts; e0 += 64) {
        t.span = span_of(p, e0 + lane);
        t.own = (t.span.end - t.span.begin + height - 1) / height;
        t.sum = running(t.own);
        t.total += __builtin_amdgcn_readlane(t.sum, 63);
    }
    return t;
}

// Tile `id` of `height` rows; no rows behind the last. An expert's tiles follow those of the experts before it.
__device__ __forceinline__ Tile tile_at(const Product& p, const Tiles& all, int id, int height) {
    if (!p.experts) {
        const int first = id * height;
        return Tile{0, first, first < p.m ? tmin(height, p.m - first) : 0};
    }
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int e0 = 0; e0 < p.experts; e0 += 64) {
        Tiles t = all;
        if (p.experts > 64) {
            t.span = span_of(p, e0 + lane);
            t.own = (t.span.end - t.span.begin + height - 1) / height;
            t.sum = running(t.own);
        }
        const uint64_t past = __ballot(before + t.sum > id);
        if (past) {
            const int at = __builtin_ctzll(past);
            const int begin = __builtin_amdgcn_readlane(t.span.begin, at), end = __builtin_amdgcn_readlane(t.span.end, at);
            const int in = id - before - (__builtin_amdgcn_readlane(t.sum, at) - __builtin_amdgcn_readlane(t.own, at));
            const int first = begin + in * height;
            return Tile{e0 + at, first, tmin(height, end - first)};
        }
        before += __builtin_amdgcn_readlane(t.sum, 63);
    }
    return Tile{0, 0, 0};
}

// The output's row of a tile's row `at`; -1 of a slot outside 0..m-1, which has none.
__device__ __forceinline__ int output_row(const Product& p, int at) {
    if (!p.experts) return at;
    const int slot = p.order[at];
    return (uint32_t)slot < (uint32_t)p.m ? slot : -1;
}
// The input's rows of N slots; one outside 0..m-1 has the first.
template <int N> __device__ __forceinline__ void input_rows(const Product& p, int* slots) {
#pragma unroll
    for (int i = 0; i < N; ++i) slots[i] = (uint32_t)slots[i] < (uint32_t)p.m ? slots[i] : 0;
    if (p.each == 1) return;
    if (p.magic) {
#pragma unroll
        for (int i = 0; i < N; ++i) slots[i] = (int)__umulhi((uint32_t)slots[i], p.magic);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) slots[i] = (int)((uint32_t)slots[i] / (uint32_t)p.each);
    }
}

}  // namespace mx
}  // namespace spa
