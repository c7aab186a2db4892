// The parts that the few-rows products share (few.hip, codes.hip): a workgroup's waves split k, each wave
// holds 16 weight rows x 16 input rows a tile as the matrix instruction leaves them (column lane & 15: the
// weight row; row 4 (lane / 16) + c: the input row), and they are joined in LDS in the order of the waves.
#pragma once

#include "dq.h"
#include "linear.h"

namespace spa {
namespace lin {
namespace {

struct FewArgs {
    Few f;
    int64_t rowbytes;
    const uint16_t* rows;     // the input rows as they lie (f.x may hold them as fragments)
};

__device__ __forceinline__ f4 mul_bf(bf8 a, bf8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
template <int KIND>
__device__ __forceinline__ f4 mul16(u4 a, u4 b, f4 c) {
    if (KIND == SRC_BF16) return mul_bf(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(hf8, a), __builtin_bit_cast(hf8, b), c, 0, 0, 0);
}

// Joins the waves' sums and writes the outputs; red has WAVES (1 + TWO) MT 256 floats. With HALVES a tile is
// 8 input rows, each as the sum of tile rows m and m + 8. again(matrix, m, n) gives a sum anew, term by
// term, where the joined one is not a number.
template <int WAVES, int MT, bool TWO, bool HALVES, class Again>
__device__ __forceinline__ void finish(const Few& f, int n0, float* red, const f4 (&acc)[1 + TWO][MT], Again again) {
    constexpr int HIGH = HALVES ? 8 : 16, S = (1 + TWO) * MT * 256;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __syncthreads();
#pragma unroll
    for (int s = 0; s <= TWO; ++s)
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c)
                red[((wave * (1 + TWO) + s) * MT + j) * 256 + (4 * (lane >> 4) + c) * 16 + (lane & 15)] = acc[s][j][c];
    __syncthreads();
    for (int i = threadIdx.x; i < MT * HIGH * 16; i += WAVES * 64) {
        const int m = i >> 4, n = n0 + (i & 15), at = HALVES ? (m >> 3) * 256 + (m & 7) * 16 + (i & 15) : i;
        if (m >= f.m || n >= f.n) continue;
        float v[1 + TWO];
#pragma unroll
        for (int s = 0; s <= TWO; ++s) {
            v[s] = 0.f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                const float* p = red + w * S + s * MT * 256 + at;
                v[s] += HALVES ? p[0] + p[128] : p[0];
            }
            if (v[s] != v[s]) v[s] = again(s, m, n);
        }
        float y;
        if constexpr (TWO) y = act_value(v[0], f.act) * v[1];
        else y = f.ex.low ? v[0] + expand(f.ex, m, n, f.n) : v[0];
        f.y[(int64_t)m * f.ldy + n] = narrow(y, f.kind);
    }
}

}  // namespace
}  // namespace lin
}  // namespace spa
