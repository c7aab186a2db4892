// Products of few 4-bit rows with 4-bit weights: the weights are read once, straight into the matrix instruction.
//
// A workgroup's waves share 16 weight rows and take 512 of k in turn; a lane reads 64 bytes of its row's codes and the four
// scales of them as one word, whose bytes the instruction picks. Which 32 of k an instruction's quarter of lanes
// holds does not matter as long as inputs and weights agree: quarter g of the lanes holds blocks 4 g + u, in
// instruction u. The waves' sums are added in LDS.
#include "../../include/seedpack_amd.h"
#include "launch.h"
#include "mx4.h"
#include "mx4_tiles.h"

namespace spa {
namespace mx {
namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
using lin::f4;
using lin::u4;

__device__ __forceinline__ v8i operand(u4 v) { return v8i{(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0}; }

// a row's 512 of k: 64 bytes of a lane's codes, and their scales; blocks behind the row's last are zeros
struct Part {
    u4 codes[4];
    uint32_t scales;
};
__device__ __forceinline__ Part load_part(const uint8_t* codes, const uint8_t* scales, int block, int pitch) {
    Part p;
    if (block < pitch) {
#pragma unroll
        for (int u = 0; u < 4; ++u) p.codes[u] = *reinterpret_cast<const u4*>(codes + (block + u) * 16);
        p.scales = *reinterpret_cast<const uint32_t*>(scales + block);
    } else {
#pragma unroll
        for (int u = 0; u < 4; ++u) p.codes[u] = u4{0, 0, 0, 0};
        p.scales = 0;
    }
    return p;
}
__device__ __forceinline__ f4 multiply(const Part& w, const Part& x, f4 acc) {
    acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(w.codes[0]), operand(x.codes[0]), acc, 4, 4, 0, (int)w.scales, 0, (int)x.scales);
    acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(w.codes[1]), operand(x.codes[1]), acc, 4, 4, 1, (int)w.scales, 1, (int)x.scales);
    acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(w.codes[2]), operand(x.codes[2]), acc, 4, 4, 2, (int)w.scales, 2, (int)x.scales);
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(w.codes[3]), operand(x.codes[3]), acc, 4, 4, 3, (int)w.scales, 3, (int)x.scales);
}

constexpr int W = 8;                                             // waves

template <bool TWO>
__global__ __launch_bounds__(W * 64) void k_few(const Product p) {
    __shared__ f4 sums[W][1 + TWO][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
    const int nt = (p.n + 15) / 16, n0 = blockIdx.x % nt * 16;
    const Tile t = tile_at(p, blockIdx.x / nt, 16);
    if (t.rows == 0) return;
    const int64_t wrow = (int64_t)t.expert * p.n + tmin(n0 + r, p.n - 1);
    const int64_t xrow = input_row(p, t.first + tmin(r, t.rows - 1));
    const uint8_t *wc = p.w0c + wrow * p.pitch * 16, *ws = p.w0s + wrow * p.pitch, *xc = p.xc + xrow * p.pitch * 16, *xs = p.xs + xrow * p.pitch;
    const uint8_t *vc = TWO ? p.w1c + wrow * p.pitch * 16 : nullptr, *vs = TWO ? p.w1s + wrow * p.pitch : nullptr;
    f4 a = {0, 0, 0, 0}, b = {0, 0, 0, 0};
    for (int k = wave * 16; k < p.pitch; k += W * 16) {
        const Part w = load_part(wc, ws, k + 4 * g, p.pitch), x = load_part(xc, xs, k + 4 * g, p.pitch);
        a = multiply(w, x, a);
        if (TWO) b = multiply(load_part(vc, vs, k + 4 * g, p.pitch), x, b);
    }
    sums[wave][0][lane] = a;
    if (TWO) sums[wave][TWO][lane] = b;
    __syncthreads();
    if (wave) return;
    for (int i = 1; i < W; ++i) {
        a += sums[i][0][lane];
        if (TWO) b += sums[i][TWO][lane];
    }
    // lane: input row r, weight rows 4 g + i
    const int64_t row = r < t.rows ? output_row(p, t.first + r) : -1;
    if (row < 0) return;
    const int64_t to = row * p.ldy + n0 + 4 * g;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (n0 + 4 * g + i >= p.n) continue;
        const float v = TWO ? lin::act_value(a[i], p.act) * b[i] : a[i];
        if (p.kind == SRC_F32) static_cast<float*>(p.y)[to + i] = v;
        else static_cast<uint16_t*>(p.y)[to + i] = lin::narrow(v, p.kind);
    }
}

}  // namespace

int product_few(const Product& p, hipStream_t st) {
    const int64_t groups = (int64_t)((p.n + 15) / 16) * most_tiles(p, 16);
    if (groups > INT32_MAX) return fail(SPA_ERR_ARG, "product: %d x %d outputs are too many", p.m, p.n);
    if (p.w1c) hipLaunchKernelGGL(k_few<true>, dim3((unsigned)groups), dim3(W * 64), 0, st, p);
    else hipLaunchKernelGGL(k_few<false>, dim3((unsigned)groups), dim3(W * 64), 0, st, p);
    SPA_HIP_TRY(hipGetLastError());
    return SPA_OK;
}

}  // namespace mx
}  // namespace spa
