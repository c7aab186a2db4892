// The parts that the few-rows products share (few.hip, codes.hip): a workgroup's waves split k, each wave
// holds 16 weight rows x 16 input rows a tile as the matrix instruction leaves them (column lane & 15: the
// weight row; row 4 (lane / 16) + c: the input row), and they are joined in LDS in the order of the waves.
#pragma once

#include "../../include/seedpack_amd.h"

#include "dq.h"
#include "launch.h"
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

// a block's bytes where they lie
struct Bytes {
    const uint8_t* p;
    __device__ __forceinline__ uint32_t u8(int k) const { return p[k]; }
    __device__ __forceinline__ uint32_t u16(int k) const { return u8(k) | (u8(k + 1) << 8); }
    __device__ __forceinline__ uint32_t u32(int k) const { return u16(k) | (u16(k + 2) << 16); }
    __device__ __forceinline__ float h(int k) const { return f16_to_f32(u16(k)); }
};
// An output's sum term by term, by a wave. Sums of codes and of offsets, or of a value's two parts, are not numbers
// where an infinity meets a code or a part of zero, or where they cancel; the sum over the weights may be infinite
// there. And with inputs near the largest number (BF16 from about 1e36) a code's base, 128 times its input, passes
// float32: the sum of codes is infinite or not a number where the sum over the weights is finite.
// A row that holds a NaN is looked through first: its sums are NaN whatever the weights are. (One lane for an output,
// weight by weight, with no such look: one row of 4096 through 12288 x 4096 Q4_K 620 us instead of 9.)
template <int T, int QK, int BS>
struct Direct {
    static constexpr bool ANEW = true;
    const FewArgs& a;
    DQ t;
    const int8_t* kv;
    __device__ __forceinline__ bool nan_in(int m) const {
        const Few& f = a.f;
        const int lane = threadIdx.x & 63;
        const uint16_t* x = a.rows + (int64_t)m * f.ldx;
        bool nan = false;
        for (int k = 8 * lane; k < f.k; k += 512) {               // rows of whole steps of 32 at 16-byte addresses
            const u4 h = *reinterpret_cast<const u4*>(x + k);
            const uint32_t top = f.kind == SRC_BF16 ? 0x7f80u : 0x7c00u;
#pragma unroll
            for (int i = 0; i < 4; ++i) nan = nan || (h[i] & 0x7fffu) > top || (h[i] >> 16 & 0x7fffu) > top;
        }
        return __ballot(nan) != 0;
    }
    __device__ __forceinline__ float operator()(int s, int m, int n) const {
        const Few& f = a.f;
        const int lane = threadIdx.x & 63;
        const uint8_t* w = (s ? f.w1 : f.w0) + (int64_t)n * a.rowbytes;
        const uint16_t* x = a.rows + (int64_t)m * f.ldx;
        float sum = 0.f;
        if constexpr (T == 1 || T == 30) {
            const int cols = (int)(a.rowbytes / 2);
            for (int k = lane; k < cols; k += 64)
                sum = fmaf(wide(x[k], f.kind), wide(reinterpret_cast<const uint16_t*>(w)[k], T == 1 ? SRC_F16 : SRC_BF16), sum);
        } else {
            for (int k = 4 * lane; k < f.k; k += 256) {
                float v[4];
                const int b = k / QK;
                dq4<T>(Bytes{w + (int64_t)b * BS}, k - b * QK, t, kv, v);
#pragma unroll
                for (int i = 0; i < 4; ++i) sum = fmaf(wide(x[k + i], f.kind), v[i], sum);
            }
        }
#pragma unroll
        for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
        return sum;
    }
};

// Joins the waves' sums and writes the outputs; red has WAVES (1 + TWO) MT 256 floats. With HALVES a tile is
// 8 input rows, each as the sum of tile rows m and m + 8. again(matrix, m, n), called by whole waves, gives a
// sum anew, term by term, where the joined one is infinite or not a number and again.nan_in(m) does not say why.
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
        const bool in = m < f.m && n < f.n;
        float v[1 + TWO];
#pragma unroll
        for (int s = 0; s <= TWO; ++s) {
            v[s] = 0.f;
            if (!in) continue;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                const float* p = red + w * S + s * MT * 256 + at;
                v[s] += HALVES ? p[0] + p[128] : p[0];
            }
        }
        if constexpr (Again::ANEW) {
            int looked = -1;
            bool nan = false;
#pragma unroll
            for (int s = 0; s <= TWO; ++s)
                for (uint64_t left = __ballot(!(fabsf(v[s]) <= 3.4028235e38f)); left; left &= left - 1) {
                    const int from = __builtin_ctzll(left), row = __builtin_amdgcn_readlane(m, from);
                    if (row != looked) nan = again.nan_in(row);
                    looked = row;
                    const float sum = nan ? __builtin_nanf("") : again(s, row, __builtin_amdgcn_readlane(n, from));
                    if (lane == from) v[s] = sum;
                }
        }
        if (!in) continue;
        float y;
        if constexpr (TWO) y = act_value(v[0], f.act) * v[1];
        else y = f.ex.low ? v[0] + expand(f.ex, m, n, f.n) : v[0];
        f.y[(int64_t)m * f.ldy + n] = narrow(y, f.kind);
    }
}

// Rows of 4096 numbers lie 8 KB apart, all in the same channel of the L2: with two or more tiles of them fetched side
// by side Q8_0 12288 x 4096 took 55 us for 32 rows. So their fragments are laid out first, 3.9 us for 32 rows of 4096 (a
// launch's latency), or by the launch of the adapters' first products. One tile is read as it lies (34.4 us for
// 151936 x 1024 with 3 rows, 36.8 by way of fragments).
__global__ __launch_bounds__(256) void k_fragments(const uint16_t* __restrict__ x, int64_t ldx, int m, Frags fr) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i < fr.tiles * (fr.k / 32) * 64) fragment(fr, x, ldx, m, i);
}
int fragments(const Few& f, const Frags& fr, hipStream_t st) {
    if (f.framed) return SPA_OK;
    const int lanes = fr.tiles * (fr.k / 32) * 64;
    hipLaunchKernelGGL(k_fragments, dim3((unsigned)((lanes + 255) / 256)), dim3(256), 0, st, f.x, f.ldx, f.m, fr);
    SPA_HIP_TRY(hipGetLastError());
    return SPA_OK;
}

}  // namespace
}  // namespace lin
}  // namespace spa
