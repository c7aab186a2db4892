// Reductions over 16, 32 or 64 neighbouring lanes whose result every lane holds, by moves between lanes that need no LDS.
#pragma once

#include "common.h"

namespace spa {

template <int CTRL> __device__ __forceinline__ uint32_t moved(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, true);
}
template <int CTRL, typename T> __device__ __forceinline__ T lane_move(T v) {
    if constexpr (sizeof(T) == 8) {
        uint64_t b;
        __builtin_memcpy(&b, &v, 8);
        b = (uint64_t)moved<CTRL>((uint32_t)(b >> 32)) << 32 | moved<CTRL>((uint32_t)b);
        __builtin_memcpy(&v, &b, 8);
    } else {
        uint32_t b;
        __builtin_memcpy(&b, &v, 4);
        b = moved<CTRL>(b);
        __builtin_memcpy(&v, &b, 4);
    }
    return v;
}
__device__ __forceinline__ double lane_xor(double v, int mask) {
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    return __longlong_as_double((long long)((uint64_t)(uint32_t)__shfl_xor((int)(b >> 32), mask) << 32 | (uint32_t)__shfl_xor((int)b, mask)));
}

// A number's two copies after rows of 16 (or 32) lanes changed places between them: the even rows' numbers everywhere, and the
// odd ones'.
template <int ROW, typename T> __device__ __forceinline__ void across_rows(T v, T& even, T& odd) {
    constexpr int N = sizeof(T) / 4;
    uint32_t b[N], c[N];
    __builtin_memcpy(b, &v, sizeof(T));
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const auto r = ROW == 16 ? __builtin_amdgcn_permlane16_swap(b[i], b[i], false, false) : __builtin_amdgcn_permlane32_swap(b[i], b[i], false, false);
        b[i] = r[0];
        c[i] = r[1];
    }
    __builtin_memcpy(&even, b, sizeof(T));
    __builtin_memcpy(&odd, c, sizeof(T));
}

// op over the L = 16, 32 or 64 lanes of a row, in an order of its own that is the same for every lane: neighbours, pairs,
// and, the pairs being alike, mirrored fours and eights, then rows of 16.
template <int L, typename T, typename F> __device__ __forceinline__ T over_row(T v, F op) {
    v = op(v, lane_move<0xb1>(v));                               // lanes 1 0 3 2
    v = op(v, lane_move<0x4e>(v));                               // lanes 2 3 0 1
    v = op(v, lane_move<0x141>(v));                              // eight lanes mirrored
    v = op(v, lane_move<0x140>(v));                              // sixteen lanes mirrored
    if constexpr (L >= 32) {
        T even, odd;
        across_rows<16>(v, even, odd);
        v = op(even, odd);
        if constexpr (L == 64) {
            across_rows<32>(v, even, odd);
            v = op(even, odd);
        }
    }
    return v;
}
template <int L, typename T> __device__ __forceinline__ T row_sum(T v) {
    return over_row<L>(v, [](T a, T b) { return a + b; });
}
template <int L, typename T> __device__ __forceinline__ T row_max(T v) {
    return over_row<L>(v, [](T a, T b) { return a > b ? a : b; });
}

}  // namespace spa
