// Dequantizers: quantized blocks -> float32, llama.cpp's dequantize_row_<type> for the 20 types of
// the path (ggml-quants.c:439-568, :961-990, :1306-1345, :1530-1550, :1732-1757, :1940-1968,
// :2489-2764). They replace the reference's k_dq_<type> launches (gpuquant.py:214-219) behind
// GPUQuant.dequantize (gpuquant.py:413-421).
//
// Mapping: a workgroup takes tiles of 4096 weights; the tile's blocks are copied to LDS with
// coalesced loads, then each lane decodes 4 consecutive outputs (every type's runs of equal header
// fields hold a multiple of 4 weights: the header is decoded once per 4 outputs, the codes read as
// one 32-bit word) and writes them as one 16-byte store. HBM-bound: 4 bytes written per weight plus
// the block bytes read once.
// Each output is the C code's expression for that element, with the same operand order (float
// products left to right, integer parts converted as the C promotions do), so the results are
// bit-identical.
#include "../../include/seedpack_amd.h"
#include "dq.h"
#include "launch.h"

namespace spa {
namespace {

// Each workgroup takes tiles of TILE weights (TILE / QK whole blocks, a multiple of 16 bytes): the
// tile's block bytes are copied to LDS with coalesced loads (16-byte loads when the source is
// 16-byte aligned, else 4- or 1-byte loads), then lane q of the tile decodes weights 4q..4q+3 from
// LDS and writes them as one 16-byte store, so consecutive lanes write consecutive bytes.
constexpr int TILE = 4096;
template <int T, int QK, int BS>
__global__ __launch_bounds__(256) void k_dq(const uint8_t* __restrict__ src, float* __restrict__ dst, int64_t nblocks,
                                            DQ t, int align) {
    constexpr int TB = TILE / QK, TBYTES = TB * BS;
    static_assert(TBYTES % 16 == 0, "tile bytes keep the source's 16-byte alignment");
    __shared__ __align__(16) uint8_t tile[TBYTES + 16];
    __shared__ int8_t kv[16];
    if (T == 20 || T == 23) {
        if (threadIdx.x < 16) kv[threadIdx.x] = KV_IQ4NL[threadIdx.x];
    }
    const int64_t ntiles = (nblocks + TB - 1) / TB;
    for (int64_t ti = blockIdx.x; ti < ntiles; ti += gridDim.x) {
        const int64_t b0 = ti * TB;
        const int nb = (int)(nblocks - b0 < TB ? nblocks - b0 : TB);
        const int bytes = nb * BS;
        const uint8_t* s = src + b0 * BS;
        __syncthreads();                     // the last tile's readers are done with it
        int done = 0;
        if (align >= 16) {
            for (int u = threadIdx.x; u < (bytes >> 4); u += 256)
                reinterpret_cast<uint4*>(tile)[u] = reinterpret_cast<const uint4*>(s)[u];
            done = bytes & ~15;
        } else if (align >= 4) {
            for (int u = threadIdx.x; u < (bytes >> 2); u += 256)
                reinterpret_cast<uint32_t*>(tile)[u] = reinterpret_cast<const uint32_t*>(s)[u];
            done = bytes & ~3;
        }
        for (int k = done + threadIdx.x; k < bytes; k += 256) tile[k] = s[k];
        __syncthreads();
        float4* out = reinterpret_cast<float4*>(dst + b0 * QK);
        for (int q = threadIdx.x; q < nb * (QK / 4); q += 256) {
            const int e = q * 4, blk = e / QK;
            float v[4];
            dq4<T>(Blk{tile, blk * BS}, e - blk * QK, t, kv, v);
            out[q] = make_float4(v[0], v[1], v[2], v[3]);
        }
    }
}

template <int T, int QK, int BS>
int run(const void* src, int64_t n, float* dst, hipStream_t st) {
    DQ t{nullptr};
    const int ti = iq_table_index(T);
    if (ti >= 0) {
        IqDeviceTable tab;
        const int rc = iq_device_table(ti, &tab, st);
        if (rc) return rc;
        t.grid = tab.grid;
    }
    const int64_t nblocks = n / QK, ntiles = (nblocks + TILE / QK - 1) / (TILE / QK);
    const uintptr_t a = reinterpret_cast<uintptr_t>(src);
    const int align = (a & 15) == 0 ? 16 : ((a & 3) == 0 ? 4 : 1);
    const int64_t grid = ntiles < 4096 ? ntiles : 4096;
    hipLaunchKernelGGL((k_dq<T, QK, BS>), dim3((unsigned)grid), dim3(256), 0, st, (const uint8_t*)src, dst, nblocks, t, align);
    SPA_HIP_TRY(hipGetLastError());
    return SPA_OK;
}

}  // namespace
}  // namespace spa

using namespace spa;

extern "C" int spa_dequantize(int type, const void* src, int64_t nrows, int64_t n_per_row, float* dst, void* stream) {
    if (nrows < 0 || n_per_row <= 0) return fail(SPA_ERR_ARG, "spa_dequantize: bad shape %lld x %lld", (long long)nrows, (long long)n_per_row);
    const int64_t n = nrows * n_per_row;
    if (n == 0) return SPA_OK;
    if (!src || !dst) return fail(SPA_ERR_ARG, "spa_dequantize: null pointer");
    if (reinterpret_cast<uintptr_t>(dst) & 15) return fail(SPA_ERR_ARG, "spa_dequantize: output not 16-byte aligned");
    hipStream_t st = (hipStream_t)stream;
#define SPA_DQ(T, QK, BS)                                                                                              \
    case T:                                                                                                            \
        if (n_per_row % QK) return fail(SPA_ERR_ARG, "spa_dequantize: row of %lld not a multiple of %d", (long long)n_per_row, QK); \
        return run<T, QK, BS>(src, n, dst, st);
    switch (type) {
        SPA_DQ(2, 32, 18) SPA_DQ(3, 32, 20) SPA_DQ(6, 32, 22) SPA_DQ(7, 32, 24) SPA_DQ(8, 32, 34)
        SPA_DQ(10, 256, 84) SPA_DQ(11, 256, 110) SPA_DQ(12, 256, 144) SPA_DQ(13, 256, 176) SPA_DQ(14, 256, 210)
        SPA_DQ(16, 256, 66) SPA_DQ(17, 256, 74) SPA_DQ(18, 256, 98) SPA_DQ(19, 256, 50) SPA_DQ(20, 32, 18)
        SPA_DQ(21, 256, 110) SPA_DQ(22, 256, 82) SPA_DQ(23, 256, 136) SPA_DQ(29, 256, 56) SPA_DQ(42, 64, 18)
        default: return fail(SPA_ERR_TYPE, "spa_dequantize: type %d not supported", type);
    }
#undef SPA_DQ
}
