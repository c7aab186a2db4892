// Products of few 4-bit rows with 4-bit weights: the weights are read once, straight into the matrix instruction.
//
// A wave takes 16 NT weight rows and 16 MT input rows, 512 of k at a time: a lane reads 64 bytes of its row's codes and the
// four scales of them as one word, whose bytes the instruction picks. Which 32 of k an instruction's quarter of lanes
// holds does not matter as long as inputs and weights agree: quarter g of the lanes holds blocks 4 g + u, in
// instruction u. (Whole lines in each load, a block a lane, need two words of scales and shifts: 8.4 us for one row of
// 12288 x 4096, not 7.4.) Of a workgroup's eight waves `split` share their rows and take the pieces of k in turn, so that a
// short row's loads are all under way at once; their sums are added in LDS.
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

// 512 of a row's k: 64 bytes of a lane's codes, and their scales
struct Part {
    u4 codes[4];
    uint32_t scales;
};
__device__ __forceinline__ Part load_part(const uint8_t* codes, const uint8_t* scales, int block) {
    Part p;
#pragma unroll
    for (int u = 0; u < 4; ++u) p.codes[u] = *reinterpret_cast<const u4*>(codes + (block + u) * 16);
    p.scales = *reinterpret_cast<const uint32_t*>(scales + block);
    return p;
}
__device__ __forceinline__ f4 multiply(const Part& w, const Part& x, f4 acc) {
    acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(w.codes[0]), operand(x.codes[0]), acc, 4, 4, 0, (int)w.scales, 0, (int)x.scales);
    acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(w.codes[1]), operand(x.codes[1]), acc, 4, 4, 1, (int)w.scales, 1, (int)x.scales);
    acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(w.codes[2]), operand(x.codes[2]), acc, 4, 4, 2, (int)w.scales, 2, (int)x.scales);
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(w.codes[3]), operand(x.codes[3]), acc, 4, 4, 3, (int)w.scales, 3, (int)x.scales);
}

constexpr int W = FEW_WAVES;

template <int MT, int NT, bool TWO>
__device__ __forceinline__ void few(const Product& p, int split) {
    constexpr int SUMS = MT * NT * (1 + TWO);
    __shared__ f4 sums[W][SUMS][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int width = W / split * 16 * NT, nt = (p.n + width - 1) / width;
    const int part = wave % split, n0 = blockIdx.x % nt * width + wave / split * 16 * NT;
    const Tile t = tile_at(p, p.experts > 64 ? Tiles{} : tiles_of(p, 16 * MT), blockIdx.x / nt, 16 * MT);
    if (t.rows == 0) return;
    const int64_t row16 = (int64_t)p.pitch * 16;
    const uint8_t *wc[NT][1 + TWO], *ws[NT][1 + TWO], *xc[MT], *xs[MT];
    int in[MT], out[MT];                                     // a lane's rows of the input and the output
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        const int64_t row = (int64_t)t.expert * p.n + tmin(n0 + 16 * i + r, p.n - 1);
        wc[i][0] = p.w0c + row * row16;
        ws[i][0] = p.w0s + row * p.pitch;
        if (TWO) {
            wc[i][TWO] = p.w1c + row * row16;
            ws[i][TWO] = p.w1s + row * p.pitch;
        }
    }
#pragma unroll
    for (int j = 0; j < MT; ++j) in[j] = out[j] = t.first + tmin(16 * j + r, t.rows - 1);
    if (p.experts) {
#pragma unroll
        for (int j = 0; j < MT; ++j) in[j] = p.order[out[j]];
#pragma unroll
        for (int j = 0; j < MT; ++j) out[j] = (uint32_t)in[j] < (uint32_t)p.m ? in[j] : -1;
        input_rows<MT>(p, in);
    }
#pragma unroll
    for (int j = 0; j < MT; ++j) {
        xc[j] = p.xc + in[j] * row16;
        xs[j] = p.xs + in[j] * (int64_t)p.pitch;
    }
    f4 acc[1 + TWO][NT][MT];
#pragma unroll
    for (int s = 0; s <= TWO; ++s)
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int j = 0; j < MT; ++j) acc[s][i][j] = f4{0, 0, 0, 0};
    for (int k = part * 16; k < p.pitch; k += split * 16) {
        // blocks behind a row's last (half of a last piece): others in their place, inputs as zeros, no scale NaN
        const int mine = k + 4 * g, block = tmin(mine, p.pitch - 4);
        const uint32_t in = mine < p.pitch ? ~0u : 0u;
        Part w[NT][1 + TWO], x[MT];
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int s = 0; s <= TWO; ++s) w[i][s] = load_part(wc[i][s], ws[i][s], block);
#pragma unroll
        for (int j = 0; j < MT; ++j) x[j] = load_part(xc[j], xs[j], block);
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int s = 0; s <= TWO; ++s) w[i][s].scales &= in;
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            x[j].scales &= in;
#pragma unroll
            for (int u = 0; u < 4; ++u) x[j].codes[u] &= in;
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int s = 0; s <= TWO; ++s) acc[s][i][j] = multiply(w[i][s], x[j], acc[s][i][j]);
        }
    }
    if (split > 1) {
#pragma unroll
        for (int s = 0; s <= TWO; ++s)
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int j = 0; j < MT; ++j) sums[wave][(s * NT + i) * MT + j][lane] = acc[s][i][j];
        __syncthreads();
    }
    // the waves of the same rows share their fragments among them
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            if ((i * MT + j) % split != part) continue;
            f4 v[1 + TWO];
#pragma unroll
            for (int s = 0; s <= TWO; ++s) {
                v[s] = acc[s][i][j];
                if (split > 1) {
                    v[s] = f4{0, 0, 0, 0};
                    for (int o = 0; o < split; ++o) v[s] += sums[wave - part + o][(s * NT + i) * MT + j][lane];
                }
            }
            // lane: input row r, weight rows 4 g + c
            const int64_t row = 16 * j + r < t.rows ? out[j] : -1;
            const int n = n0 + 16 * i + 4 * g;
            if (row < 0 || n >= p.n) continue;
            const int64_t to = row * p.ldy + n;
            if (TWO) {
#pragma unroll
                for (int c = 0; c < 4; ++c) v[0][c] = lin::act_value(v[0][c], p.act) * v[TWO][c];
            }
            if (p.kind == SRC_F32) {
                float* const y = static_cast<float*>(p.y) + to;
                if (n + 4 <= p.n) {
                    __builtin_memcpy(y, &v[0], 16);               // at any number's address
                } else {
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        if (n + c < p.n) y[c] = v[0][c];
                }
            } else {
                uint16_t* const y = static_cast<uint16_t*>(p.y) + to;
                const lin::u2 h = {lin::narrow2(v[0][0], v[0][1], p.kind), lin::narrow2(v[0][2], v[0][3], p.kind)};
                if (n + 4 <= p.n) {
                    __builtin_memcpy(y, &h, 8);
                } else {
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        if (n + c < p.n) y[c] = (uint16_t)(h[c >> 1] >> (16 * (c & 1)));
                }
            }
        }
}

template <int MT, int NT, bool TWO>
__global__ __launch_bounds__(W * 64) void k_few(const Product p, int split) {
    few<MT, NT, TWO>(p, split);
}

template <int MT, int NT, bool TWO> int launch(const Product& p, hipStream_t st) {
    const int split = few_split(p.pitch);
    const int width = W / split * 16 * NT;
    const int64_t groups = (int64_t)((p.n + width - 1) / width) * most_tiles(p, 16 * MT);
    if (!one_launch(groups, W * 64)) return fail(SPA_ERR_ARG, "product: %d x %d outputs are too many", p.m, p.n);
    hipLaunchKernelGGL((k_few<MT, NT, TWO>), dim3((unsigned)groups), dim3(W * 64), 0, st, p, split);
    SPA_HIP_TRY(hipGetLastError());
    return SPA_OK;
}

}  // namespace

int product_few(const Product& p, bool wide, hipStream_t st) {
    if (wide) return launch<2, 2, false>(p, st);
    return p.w1c ? launch<1, 1, true>(p, st) : launch<1, 1, false>(p, st);
}

}  // namespace mx
}  // namespace spa
