// The passes over rows around the products of gemm.hip: operands brought into the form that it takes
// (padded, converted, transposed), the powers of two that conversions take out, and the adapters' first
// product. All but the last are bound by memory.
#include "../../include/seedpack_amd.h"
#include "dq.h"
#include "launch.h"
#include "linear.h"

namespace spa {
namespace lin {
namespace {

// eight elements from k on, zeros from n on; wide: the address is 16-byte aligned wherever k + 8 <= n
__device__ __forceinline__ void load8(const uint16_t* row, int64_t k, int64_t n, bool wide8, uint16_t (&h)[8]) {
    if (wide8 && k + 8 <= n) {
        *reinterpret_cast<u4*>(h) = *reinterpret_cast<const u4*>(row + k);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = k + i < n ? row[k + i] : 0;
}

__global__ __launch_bounds__(256) void k_pack(const uint16_t* __restrict__ src, int64_t ld, int64_t rows, int64_t k,
                                              uint16_t* __restrict__ dst, int64_t kp, bool wide8) {
    const int64_t per = kp / 8, total = rows * per;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
        const int64_t r = i / per, c = (i - r * per) * 8;
        __align__(16) uint16_t h[8];
        load8(src + r * ld, c, k, wide8, h);
        *reinterpret_cast<u4*>(dst + r * kp + c) = *reinterpret_cast<u4*>(h);
    }
}

// a workgroup's largest or total float, the same in every lane; in an order of its own shape only
template <bool MAX>
__device__ __forceinline__ float reduce256(float v, float* lds) {
#pragma unroll
    for (int s = 32; s; s >>= 1) {
        const float o = __shfl_xor(v, s);
        v = MAX ? fmaxf(v, o) : v + o;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    return MAX ? fmaxf(fmaxf(lds[0], lds[1]), fmaxf(lds[2], lds[3])) : (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

__device__ __forceinline__ float size_of(float v) {              // |v|, zero for infinities and NaN
    const float a = fabsf(v);
    return a <= 3.4028235e38f ? a : 0.f;
}
// the power of two that brings values up to `top` below 2^15
__device__ __forceinline__ int exponent_for(float top) {
    if (!(top > 0.f)) return 0;
    int e;
    frexpf(top, &e);
    return e - 15;
}
__global__ __launch_bounds__(256) void k_half_rows(const uint16_t* __restrict__ src, int kind, int64_t ld, int64_t k,
                                                   uint16_t* __restrict__ dst, int64_t kp, int32_t* __restrict__ e_out,
                                                   float* __restrict__ norm, bool wide8) {
    __shared__ float lds[4];
    const int64_t row = blockIdx.x;
    src += row * ld;
    dst += row * kp;
    float most = 0.f;
    for (int64_t c = threadIdx.x * 8; c < k; c += 2048) {
        __align__(16) uint16_t h[8];
        load8(src, c, k, wide8, h);
#pragma unroll
        for (int i = 0; i < 8; ++i) most = fmaxf(most, size_of(wide(h[i], kind)));
    }
    const int e = exponent_for(reduce256<true>(most, lds));
    float sum = 0.f;
    for (int64_t c = threadIdx.x * 8; c < kp; c += 2048) {
        __align__(16) uint16_t h[8];
        load8(src, c, k, wide8, h);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float v = ldexpf(wide(h[i], kind), -e);
            sum = fmaf(size_of(v), size_of(v), sum);
            h[i] = narrow(v, SRC_F16);
        }
        *reinterpret_cast<u4*>(dst + c) = *reinterpret_cast<u4*>(h);
    }
    if (threadIdx.x == 0) e_out[row] = e;
    if (norm) {
        sum = reduce256<false>(sum, lds);
        if (threadIdx.x == 0) norm[row] = fminf(ldexpf(sqrtf(sum), e), 3e38f);
    }
}

// what a block's weights are at most in size, by its header: scale (and offset) times the largest code.
// It is up to 2^10 over the largest weight itself: binary16 has 39 binary orders below 2^15.
template <int T>
__device__ __forceinline__ float block_bound(const uint8_t* b) {
    auto h = [&](int k) { return size_of(f16_to_f32((uint32_t)b[k] | ((uint32_t)b[k + 1] << 8))); };
    switch (T) {
        case 2: return 8.f * h(0);
        case 3: return 15.f * h(0) + h(2);
        case 6: return 16.f * h(0);
        case 7: return 31.f * h(0) + h(2);
        case 8: return 128.f * h(0);
        case 42: return 2.f * h(0);
        case 10: return 45.f * h(80) + 15.f * h(82);
        case 11: return 128.f * h(108);
        case 12: return 945.f * h(0) + 63.f * h(2);
        case 13: return 1953.f * h(0) + 63.f * h(2);
        case 14: return 4096.f * h(208);
        case 16: case 17: case 22: return 167.f * h(0);
        case 18: return 481.f * h(0);
        case 21: return 465.f * h(0);
        case 19: return 17.f * h(0);
        case 29: {
            const uint32_t sf = (uint32_t)(b[49] >> 4) | (uint32_t)(b[51] & 0xf0) | ((uint32_t)(b[53] & 0xf0) << 4) |
                                ((uint32_t)(b[55] & 0xf0) << 8);
            return 17.f * size_of(f16_to_f32(sf));
        }
        case 20: return 127.f * h(0);
        default: return 4064.f * h(0);                            // 23
    }
}

constexpr int TILE = 4096;
template <int T, int QK, int BS>
__global__ __launch_bounds__(256) void k_half_blocks(const uint8_t* __restrict__ src, int64_t k, uint16_t* __restrict__ dst,
                                                     int64_t kp, int32_t* __restrict__ e_out, float* __restrict__ norm, DQ t,
                                                     int align) {
    constexpr int TB = TILE / QK, TBYTES = TB * BS;
    __shared__ __align__(16) uint8_t tile[TBYTES + 16];
    __shared__ int8_t kv[16];
    __shared__ float lds[4];
    if (T == 20 || T == 23) {
        if (threadIdx.x < 16) kv[threadIdx.x] = KV_IQ4NL[threadIdx.x];
    }
    const int64_t row = blockIdx.x, nb = k / QK;
    src += row * nb * BS;
    dst += row * kp;
    float most = 0.f;
    for (int64_t b = threadIdx.x; b < nb; b += 256) most = fmaxf(most, block_bound<T>(src + b * BS));
    const int e = exponent_for(reduce256<true>(most, lds));
    float sum = 0.f;
    for (int64_t b0 = 0; b0 < nb; b0 += TB) {
        const int n = (int)(nb - b0 < TB ? nb - b0 : TB), bytes = n * BS;
        const uint8_t* s = src + b0 * BS;
        __syncthreads();
        int done = 0;
        if (align >= 16) {
            for (int u = threadIdx.x; u < (bytes >> 4); u += 256)
                reinterpret_cast<u4*>(tile)[u] = reinterpret_cast<const u4*>(s)[u];
            done = bytes & ~15;
        } else if (align >= 4) {
            for (int u = threadIdx.x; u < (bytes >> 2); u += 256)
                reinterpret_cast<uint32_t*>(tile)[u] = reinterpret_cast<const uint32_t*>(s)[u];
            done = bytes & ~3;
        } else if (align >= 2) {
            for (int u = threadIdx.x; u < (bytes >> 1); u += 256)
                reinterpret_cast<uint16_t*>(tile)[u] = reinterpret_cast<const uint16_t*>(s)[u];
            done = bytes & ~1;
        }
        for (int u = done + threadIdx.x; u < bytes; u += 256) tile[u] = s[u];
        __syncthreads();
        for (int q = threadIdx.x; q < n * (QK / 4); q += 256) {
            const int o = q * 4, blk = o / QK;
            float v[4];
            dq4<T>(Blk{tile, blk * BS}, o - blk * QK, t, kv, v);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = ldexpf(v[i], -e);
                sum = fmaf(size_of(v[i]), size_of(v[i]), sum);
            }
            *reinterpret_cast<u2*>(dst + b0 * QK + o) = u2{narrow2(v[0], v[1], SRC_F16), narrow2(v[2], v[3], SRC_F16)};
        }
    }
    for (int64_t c = k + threadIdx.x; c < kp; c += 256) dst[c] = 0;
    if (threadIdx.x == 0) e_out[row] = e;
    if (norm) {
        sum = reduce256<false>(sum, lds);
        if (threadIdx.x == 0) norm[row] = fminf(ldexpf(sqrtf(sum), e), 3e38f);
    }
}

// 64 x 64 tiles through LDS: read along a row's columns, written along a column's rows
__global__ __launch_bounds__(256) void k_transpose(const uint16_t* __restrict__ src, int64_t ld, int64_t rows, int64_t cols,
                                                   uint16_t* __restrict__ dst, int64_t ldd, int64_t rp, int64_t tiles_c) {
    __shared__ uint16_t t[64][66];
    const int64_t r0 = blockIdx.x / tiles_c * 64, c0 = blockIdx.x % tiles_c * 64;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int u = i * 256 + threadIdx.x, r = u >> 5, c = (u & 31) * 2;
        const int64_t R = r0 + r, C = c0 + c;
        uint16_t a = 0, b = 0;
        if (R < rows && C < cols) a = src[R * ld + C];
        if (R < rows && C + 1 < cols) b = src[R * ld + C + 1];
        t[r][c] = a;
        t[r][c + 1] = b;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int u = i * 256 + threadIdx.x, c = u >> 5, r = (u & 31) * 2;
        const int64_t R = r0 + r, C = c0 + c;
        if (C < cols && R < rp)                                   // rp is even
            *reinterpret_cast<uint32_t*>(dst + C * ldd + R) = (uint32_t)t[r][c] | ((uint32_t)t[r + 1][c] << 16);
    }
}

// the largest 2-norm and the largest power of two of both matrices' rows
struct Top {
    float norm;
    int32_t e;
};
__global__ __launch_bounds__(1024) void k_top(const float* n0, const int32_t* e0, const float* n1, const int32_t* e1, int64_t n, Top* top) {
    __shared__ float ln[16];
    __shared__ int le[16];
    float a = 0.f;
    int e = INT32_MIN;
    for (int64_t i = threadIdx.x; i < n; i += 1024) {
        a = fmaxf(a, fmaxf(n0[i], n1[i]));
        e = tmax(e, tmax(e0[i], e1[i]));
    }
#pragma unroll
    for (int s = 32; s; s >>= 1) {
        a = fmaxf(a, __shfl_xor(a, s));
        e = tmax(e, __shfl_xor(e, s));
    }
    if ((threadIdx.x & 63) == 0) {
        ln[threadIdx.x >> 6] = a;
        le[threadIdx.x >> 6] = e;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 16; ++w) {
            a = fmaxf(a, ln[w]);
            e = tmax(e, le[w]);
        }
        *top = Top{a, e};
    }
}

// |dh u act'(g)| and |dh act(g)| are at most 1.13 |dh| |x_m| |w_n| (Cauchy-Schwarz; |act'| <= 1.13,
// |act(g)| <= |g|). Their row is multiplied by the weights' powers of two, so the largest of those counts too.
__global__ __launch_bounds__(256) void k_grad_exponents(const uint16_t* __restrict__ dh, int kind, int64_t ld, int64_t n,
                                                        const float* __restrict__ xnorm, const Top* __restrict__ top,
                                                        int32_t* __restrict__ e) {
    __shared__ float lds[4];
    const int64_t row = blockIdx.x;
    float most = 0.f;
    for (int64_t c = threadIdx.x; c < n; c += 256) most = fmaxf(most, size_of(wide(dh[row * ld + c], kind)));
    most = reduce256<true>(most, lds);
    if (threadIdx.x) return;
    const float a = xnorm[row], b = top->norm;
    if (!(most > 0.f) || !(a > 0.f) || !(b > 0.f)) {
        e[row] = 0;
        return;
    }
    int em, ea, eb;
    frexpf(most, &em);
    frexpf(a, &ea);
    frexpf(b, &eb);
    e[row] = em + ea + eb + 1 + top->e - 15;
}

__global__ void k_zero_rows(uint16_t* p, int64_t ld, int64_t rows, int64_t k) {
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < rows * k; i += gridDim.x * 256ll) p[i / k * ld + i % k] = 0;
}

// low[m][r] = s_a sum_k x[m][k] A_a[r][k] for 16 rows a workgroup and one adapter: gridDim.y workgroups
// take the adapters among the 16 rows in turn, in rising order, most of them finding none. The whole tile is
// multiplied by the adapter's matrix and its own rows are kept. Each of 8 waves takes every eighth step of
// 32 k, two steps at a time so that ten loads are under way; 64 ranks at a time, so that x is read once for
// the usual ranks.
constexpr int LOW_WAVES = 8;
template <int KIND, bool WIDE>
__global__ __launch_bounds__(LOW_WAVES * 64) void k_low(const uint16_t* __restrict__ x, int64_t ldx, int64_t m, int64_t k,
                                                        const uint16_t* __restrict__ a_all, const float* __restrict__ scale,
                                                        const int32_t* __restrict__ which, int pool, int rank,
                                                        float* __restrict__ low, int rp, bool wide_x, bool wide_a) {
    __shared__ float part[LOW_WAVES][4][256];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t m0 = (int64_t)blockIdx.x * 16;
    const int row = lane & 15, kc = (lane >> 4) * 8;
    const int mine = m0 + row < m ? which[m0 + row] : -1;
    const uint16_t* xr = x + (m0 + row < m ? m0 + row : m - 1) * ldx;
    if (blockIdx.y == 0) {                                        // rows without an adapter: zeros
        for (int i = threadIdx.x; i < 16 * rp; i += LOW_WAVES * 64) {
            const int64_t mi = m0 + i / rp;
            if (mi < m) {
                const int a = which[mi];
                if (a < 0 || a >= pool) low[mi * rp + i % rp] = 0.f;
            }
        }
    }
    int a = -1;
    for (unsigned turn = 0;; ++turn) {                            // the same in every lane and wave
        int best = mine > a && mine < pool ? mine : INT32_MAX;
#pragma unroll
        for (int s = 8; s; s >>= 1) best = tmin(best, __shfl_xor(best, s));
        a = __builtin_amdgcn_readfirstlane(best);
        if (a == INT32_MAX) return;
        if (turn == blockIdx.y) break;
    }
    const uint16_t* aa = a_all + (int64_t)a * rank * k;
    for (int r0 = 0; r0 < rp; r0 += 64) {
        const int tiles = tmin(4, (rp - r0) / 16);
        const uint16_t* ar[4];
        f4 acc[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int r = r0 + 16 * j + row;                      // ranks beyond the last take its row: they are not kept
            ar[j] = aa + (int64_t)(r < rank ? r : rank - 1) * k;
            acc[j] = f4{0, 0, 0, 0};
        }
        auto fetch = [&](int64_t k0, u4& xv, u4 (&av)[4]) {
            if (WIDE) {                                           // rows of whole steps at 16-byte addresses
                const bool in = k0 < k;
                xv = in ? *reinterpret_cast<const u4*>(xr + k0 + kc) : u4{0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    av[j] = in && j < tiles ? *reinterpret_cast<const u4*>(ar[j] + k0 + kc) : u4{0, 0, 0, 0};
            } else {
                __align__(16) uint16_t h[8];
                load8(xr, k0 + kc, k, wide_x, h);
                xv = *reinterpret_cast<u4*>(h);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (j < tiles) load8(ar[j], k0 + kc, k, wide_a, h);
                    av[j] = *reinterpret_cast<u4*>(h);
                }
            }
        };
        auto mul = [&](u4 xv, const u4 (&av)[4]) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (j >= tiles) break;
                if (KIND == SRC_BF16)
                    acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, xv), __builtin_bit_cast(bf8, av[j]), acc[j], 0, 0, 0);
                else
                    acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(hf8, xv), __builtin_bit_cast(hf8, av[j]), acc[j], 0, 0, 0);
            }
        };
        constexpr int STEP = LOW_WAVES * 32;
        u4 x0, x1, a0[4], a1[4];
        fetch(wave * 32, x0, a0);
        fetch(wave * 32 + STEP, x1, a1);
        for (int64_t k0 = wave * 32; k0 < k; k0 += 2 * STEP) {
            u4 x2, x3, a2[4], a3[4];
            fetch(k0 + 2 * STEP, x2, a2);
            fetch(k0 + 3 * STEP, x3, a3);
            mul(x0, a0);
            mul(x1, a1);
            x0 = x2;
            x1 = x3;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                a0[j] = a2[j];
                a1[j] = a3[j];
            }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) part[wave][j][(4 * (lane >> 4) + c) * 16 + row] = acc[j][c];
        __syncthreads();
        for (int i = threadIdx.x; i < 1024; i += LOW_WAVES * 64) {
            const int j = i >> 8, mr = (i >> 4) & 15, r = r0 + 16 * j + (i & 15);
            const int64_t mi = m0 + mr;
            if (mi < m && r < rp && which[mi] == a) {
                float v = 0.f;
#pragma unroll
                for (int w = 0; w < LOW_WAVES; ++w) v += part[w][j][i & 255];
                low[mi * rp + r] = r < rank ? scale[a] * v : 0.f;
            }
        }
    }
}

bool aligned8(const void* p, int64_t ld) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % 8 == 0; }

}  // namespace

int pack_rows(const uint16_t* src, int64_t ld, int64_t rows, int64_t k, uint16_t* dst, int64_t kp, hipStream_t st) {
    const int64_t groups = (rows * (kp / 8) + 255) / 256;
    hipLaunchKernelGGL(k_pack, dim3((unsigned)(groups < 8192 ? groups : 8192)), dim3(256), 0, st, src, ld, rows, k, dst, kp,
                       aligned8(src, ld));
    SPA_HIP_TRY(hipGetLastError());
    return SPA_OK;
}

int half_rows(const uint16_t* src, int kind, int64_t ld, int64_t rows, int64_t k, uint16_t* dst, int64_t kp, int32_t* e,
              float* norm, hipStream_t st) {
    hipLaunchKernelGGL(k_half_rows, dim3((unsigned)rows), dim3(256), 0, st, src, kind, ld, k, dst, kp, e, norm, aligned8(src, ld));
    SPA_HIP_TRY(hipGetLastError());
    return SPA_OK;
}

int half_blocks(int type, const uint8_t* src, int64_t rows, int64_t k, uint16_t* dst, int64_t kp, int32_t* e, float* norm,
                hipStream_t st) {
    DQ t{nullptr};
    const int ti = iq_table_index(type);
    if (ti >= 0) {
        IqDeviceTable tab;
        const int rc = iq_device_table(ti, &tab, st);
        if (rc) return rc;
        t.grid = tab.grid;
    }
    const uintptr_t a = reinterpret_cast<uintptr_t>(src) | (uintptr_t)(k / type_qk(type) * type_bs(type));
    const int align = (a & 15) == 0 ? 16 : ((a & 3) == 0 ? 4 : ((a & 1) == 0 ? 2 : 1));
    switch (type) {
#define SPA_BLOCKS(T, QK, BS)                                                                                           \
    case T:                                                                                                             \
        hipLaunchKernelGGL((k_half_blocks<T, QK, BS>), dim3((unsigned)rows), dim3(256), 0, st, src, k, dst, kp, e, norm, t, align); \
        break;
        SPA_BLOCKS(2, 32, 18) SPA_BLOCKS(3, 32, 20) SPA_BLOCKS(6, 32, 22) SPA_BLOCKS(7, 32, 24) SPA_BLOCKS(8, 32, 34)
        SPA_BLOCKS(10, 256, 84) SPA_BLOCKS(11, 256, 110) SPA_BLOCKS(12, 256, 144) SPA_BLOCKS(13, 256, 176) SPA_BLOCKS(14, 256, 210)
        SPA_BLOCKS(16, 256, 66) SPA_BLOCKS(17, 256, 74) SPA_BLOCKS(18, 256, 98) SPA_BLOCKS(19, 256, 50) SPA_BLOCKS(20, 32, 18)
        SPA_BLOCKS(21, 256, 110) SPA_BLOCKS(22, 256, 82) SPA_BLOCKS(23, 256, 136) SPA_BLOCKS(29, 256, 56) SPA_BLOCKS(42, 64, 18)
#undef SPA_BLOCKS
        default: return fail(SPA_ERR_TYPE, "weights of type %d are not supported", type);
    }
    SPA_HIP_TRY(hipGetLastError());
    return SPA_OK;
}

int transpose16(const uint16_t* src, int64_t ld, int64_t rows, int64_t cols, uint16_t* dst, int64_t ldd, int64_t rp,
                hipStream_t st) {
    const int64_t tr = (rp + 63) / 64, tc = (cols + 63) / 64;
    hipLaunchKernelGGL(k_transpose, dim3((unsigned)(tr * tc)), dim3(256), 0, st, src, ld, rows, cols, dst, ldd, rp, tc);
    SPA_HIP_TRY(hipGetLastError());
    return SPA_OK;
}

int grad_exponents(const uint16_t* dh, int kind, int64_t ld, int64_t rows, int64_t n, const float* xnorm, const float* n0,
                   const int32_t* e0, const float* n1, const int32_t* e1, void* top, int32_t* e, hipStream_t st) {
    hipLaunchKernelGGL(k_top, dim3(1), dim3(1024), 0, st, n0, e0, n1, e1, n, (Top*)top);
    SPA_HIP_TRY(hipGetLastError());
    hipLaunchKernelGGL(k_grad_exponents, dim3((unsigned)rows), dim3(256), 0, st, dh, kind, ld, n, xnorm, (const Top*)top, e);
    SPA_HIP_TRY(hipGetLastError());
    return SPA_OK;
}

int zero_rows(uint16_t* p, int64_t ld, int64_t rows, int64_t k, hipStream_t st) {
    const int64_t groups = (rows * k + 255) / 256;
    hipLaunchKernelGGL(k_zero_rows, dim3((unsigned)(groups < 4096 ? groups : 4096)), dim3(256), 0, st, p, ld, rows, k);
    SPA_HIP_TRY(hipGetLastError());
    return SPA_OK;
}

int low_rows(const uint16_t* x, int64_t ldx, int kind, int64_t m, int64_t k, const uint16_t* a, const float* scale,
             const int32_t* which, int pool, int rank, float* low, int rp, hipStream_t st) {
    const dim3 grid((unsigned)((m + 15) / 16), (unsigned)(pool < 16 ? pool : 16)), block(LOW_WAVES * 64);
    const bool wx = aligned8(x, ldx), wa = aligned8(a, k), whole = wx && wa && k % 32 == 0;
#define SPA_LOW(KIND, WIDE) \
    hipLaunchKernelGGL((k_low<KIND, WIDE>), grid, block, 0, st, x, ldx, m, k, a, scale, which, pool, rank, low, rp, wx, wa)
    if (kind == SRC_BF16) {
        if (whole) SPA_LOW(SRC_BF16, true);
        else SPA_LOW(SRC_BF16, false);
    } else {
        if (whole) SPA_LOW(SRC_F16, true);
        else SPA_LOW(SRC_F16, false);
    }
#undef SPA_LOW
    SPA_HIP_TRY(hipGetLastError());
    return SPA_OK;
}

}  // namespace lin
}  // namespace spa
