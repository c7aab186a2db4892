// The many-rows product of 16-bit operands, sum_k x[m][k] w[n][k], with what follows it in the same
// launch: the adapters' second product, or the gated block's activation and product, or its gradient.
//
// A workgroup computes TN weight rows x TM input rows. Both operands are contiguous along k, so a tile
// step of 64 k is TN + TM rows of 128 bytes; they go from HBM / L2 straight to LDS (16-byte
// global_load_lds) into one of two buffers while the other is multiplied. LDS rows are 128 bytes too,
// their eight 16-byte chunks stored at chunk ^ (row & 7): a fragment read takes the same chunk of 8
// consecutive rows in a phase, which the exchange spreads over all banks. The exchange is made on the
// global side (a lane fetches the chunk that belongs at its place).
// Weights are the matrix instruction's first operand: a lane then holds four consecutive n of one input
// row, which leave as one 8-byte store.
// For the gated forms half of the TN rows are the gate's and half the same rows of the up projection, so
// that one lane holds both values of an output.
#include "../../include/seedpack_amd.h"
#include "launch.h"
#include "linear.h"

namespace spa {
namespace lin {
namespace {

constexpr int BK = 64;

template <int HALF> struct Op;
template <> struct Op<SRC_BF16> {
    static __device__ __forceinline__ f16v mul(u4 a, u4 b, f16v c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
    }
};
template <> struct Op<SRC_F16> {
    static __device__ __forceinline__ f16v mul(u4 a, u4 b, f16v c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(hf8, a), __builtin_bit_cast(hf8, b), c, 0, 0, 0);
    }
};
__device__ __forceinline__ f16v mul_bf(bf8 a, bf8 b, f16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

typedef const __attribute__((address_space(1))) void* gptr;
typedef __attribute__((address_space(3))) void* lptr;

// the least adapter number above `after` among the tile's rows, or INT32_MAX
template <int TM>
__device__ __forceinline__ int next_adapter(const Expand& ex, int m0, int m, int after) {
    int best = INT32_MAX;
    for (int r = threadIdx.x & 63; r < TM; r += 64) {
        if (m0 + r >= m) continue;
        const int a = ex.which[m0 + r];
        if (a > after && a < ex.pool && a < best) best = a;
    }
#pragma unroll
    for (int s = 32; s; s >>= 1) best = tmin(best, __shfl_xor(best, s));
    return best;
}

template <int HALF, int TN, int TM, int WN, int WM, int OUT>
__global__ __launch_bounds__(WN * WM * 64) void k_gemm(const Gemm g) {
    constexpr int NW = WN * WM;                              // waves
    constexpr bool TWO = OUT != OUT_PLAIN;
    constexpr int TNE = TWO ? TN / 2 : TN;                   // output columns of the tile
    constexpr int FN = TN / WN / 32, FM = TM / WM / 32;      // 32 x 32 fragments of a wave
    constexpr int LOADS = (TN + TM) / 8 / NW;                // 8 rows by one load of a wave
    static_assert((TN + TM) % (8 * NW) == 0 && (!TWO || FN % 2 == 0), "tile shape");
    __shared__ __align__(16) uint16_t tile[2][(TN + TM) * BK];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // Tiles are dealt so that each of the 8 XCDs, which take workgroups in turn, has a run of neighbours
    // (its L2 then serves their shared rows), and a run covers 8 tiles of input rows per tile of weights.
    const int nt = (g.n + TNE - 1) / TNE, mt = (g.m + TM - 1) / TM, total = nt * mt;
    int id = blockIdx.x;
    {
        const int q = total / 8, r = total % 8, xcd = id & 7, at = id >> 3;
        id = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + at;
    }
    constexpr int GROUP = 8;
    const int band = id / (GROUP * nt), in = id - band * GROUP * nt;
    const int height = tmin(GROUP, mt - band * GROUP);
    const int m0 = (band * GROUP + in % height) * TM, n0 = in / height * TNE;

    // where this lane fetches from: row lane / 8 of an 8-row load, the chunk that belongs at its place
    const char* base[LOADS];
    uint32_t off[LOADS];
    const int lr = lane >> 3, chunk = (lane & 7) ^ lr;
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
        const int r0 = (j * NW + wave) * 8;
        if (r0 < TN) {
            const bool second = TWO && r0 >= TNE;
            const int r = tmin(n0 + r0 - (second ? TNE : 0) + lr, g.n - 1) - n0;
            base[j] = reinterpret_cast<const char*>((second ? g.w1 : g.w0) + (int64_t)n0 * g.ldw);
            off[j] = (uint32_t)r * (uint32_t)(2 * g.ldw) + 16 * chunk;
        } else {
            const int r = tmin(m0 + r0 - TN + lr, g.m - 1) - m0;
            base[j] = reinterpret_cast<const char*>(g.x + (int64_t)m0 * g.ldx);
            off[j] = (uint32_t)r * (uint32_t)(2 * g.ldx) + 16 * chunk;
        }
    }
    auto fetch = [&](int buf, int kt) {
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const char* p = base[j] + (int64_t)kt * (2 * BK);
            __builtin_amdgcn_global_load_lds((gptr)(p + off[j]), (lptr)(&tile[buf][(j * NW + wave) * 8 * BK]), 16, 0, 0);
        }
    };

    const int wn = wave % WN, wm = wave / WN;
    const int fr = lane & 31, fk = lane >> 5;                // a fragment's row and its half of 16 k
    int arow[FN], brow[FM];
#pragma unroll
    for (int i = 0; i < FN; ++i) {
        if (TWO) arow[i] = (i < FN / 2 ? 0 : TNE) + wn * (TNE / WN) + (i % (FN / 2)) * 32 + fr;
        else arow[i] = wn * (TN / WN) + i * 32 + fr;
    }
#pragma unroll
    for (int i = 0; i < FM; ++i) brow[i] = TN + wm * (TM / WM) + i * 32 + fr;

    f16v acc[FN][FM];
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j)
#pragma unroll
            for (int c = 0; c < 16; ++c) acc[i][j][c] = 0.f;

    const int steps = g.k / BK;
    fetch(0, 0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    for (int kt = 0; kt < steps; ++kt) {
        const uint16_t* t = tile[kt & 1];
        // the other buffer's last readers passed the barrier at the end of the step before
        if (kt + 1 < steps) fetch((kt + 1) & 1, kt + 1);
#pragma unroll
        for (int kk = 0; kk < BK / 16; ++kk) {
            u4 a[FN], b[FM];
#pragma unroll
            for (int i = 0; i < FN; ++i)
                a[i] = *reinterpret_cast<const u4*>(t + arow[i] * BK + (((2 * kk + fk) ^ (arow[i] & 7)) * 8));
#pragma unroll
            for (int i = 0; i < FM; ++i)
                b[i] = *reinterpret_cast<const u4*>(t + brow[i] * BK + (((2 * kk + fk) ^ (brow[i] & 7)) * 8));
#pragma unroll
            for (int i = 0; i < FN; ++i)
#pragma unroll
                for (int j = 0; j < FM; ++j) acc[i][j] = Op<HALF>::mul(a[i], b[j], acc[i][j]);
        }
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
    }

    // lane: input row (lane & 31) of a fragment; register 4 q + c: weight row 8 q + 4 (lane >> 5) + c
    const int nw = n0 + wn * (TNE / WN) + 4 * fk;
    const bool vec = OUT == OUT_GRAD || ((g.ldy & 3) == 0 && (reinterpret_cast<uintptr_t>(g.y) & 7) == 0);
    if constexpr (OUT == OUT_PLAIN) {
        if (g.xe || g.we0) {
#pragma unroll
            for (int j = 0; j < FM; ++j) {
                const int mi = m0 + brow[j] - TN;
                const int xe = g.xe && mi < g.m ? g.xe[mi] : 0;
#pragma unroll
                for (int i = 0; i < FN; ++i)
#pragma unroll
                    for (int c = 0; c < 16; ++c) {
                        const int ni = nw + 32 * i + 8 * (c >> 2) + (c & 3);
                        acc[i][j][c] = ldexpf(acc[i][j][c], xe + (g.we0 && ni < g.n ? g.we0[ni] : 0));
                    }
            }
        }
        if (g.ex.low) {
            // the adapters' second product, one adapter of the tile's rows at a time: rows of another
            // adapter take part with zeros. low is split into two BF16 parts, b into two where it is F16.
            const Expand& ex = g.ex;
            for (int a = next_adapter<TM>(ex, m0, g.m, -1); a != INT32_MAX; a = next_adapter<TM>(ex, m0, g.m, a)) {
                const uint16_t* ba = ex.b + (int64_t)a * g.n * ex.rank;
                for (int r0 = 0; r0 < ex.rp; r0 += 16) {
                    const int r = r0 + 8 * fk;
                    bf8 zh[FM], zl[FM];
#pragma unroll
                    for (int j = 0; j < FM; ++j) {
                        const int mi = m0 + brow[j] - TN;
                        float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
                        if (mi < g.m && ex.which[mi] == a) {
                            const f4* z = reinterpret_cast<const f4*>(ex.low + (int64_t)mi * ex.rp + r);
#pragma unroll
                            for (int c = 0; c < 8; ++c) v[c] = z[c >> 2][c & 3];
                        }
                        split8(v, zh[j], zl[j]);
                    }
#pragma unroll
                    for (int i = 0; i < FN; ++i) {
                        const int ni = n0 + arow[i];
                        uint16_t h[8] = {0, 0, 0, 0, 0, 0, 0, 0};
                        if (ni < g.n && r < ex.rank) {
                            const uint16_t* p = ba + (int64_t)ni * ex.rank + r;
                            if (ex.wide_b) {
                                *reinterpret_cast<u4*>(h) = *reinterpret_cast<const u4*>(p);
                            } else {
#pragma unroll
                                for (int c = 0; c < 8; ++c)
                                    if (r + c < ex.rank) h[c] = p[c];
                            }
                        }
                        bf8 bh, bl;
                        if (ex.kind == SRC_BF16) {
                            bh = __builtin_bit_cast(bf8, *reinterpret_cast<u4*>(h));
                        } else {
                            float v[8];
#pragma unroll
                            for (int c = 0; c < 8; ++c) v[c] = wide(h[c], SRC_F16);
                            split8(v, bh, bl);
                        }
#pragma unroll
                        for (int j = 0; j < FM; ++j) {
                            acc[i][j] = mul_bf(bh, zl[j], acc[i][j]);
                            if (ex.kind != SRC_BF16) acc[i][j] = mul_bf(bl, zh[j], acc[i][j]);
                            acc[i][j] = mul_bf(bh, zh[j], acc[i][j]);
                        }
                    }
                }
            }
        }
#pragma unroll
        for (int j = 0; j < FM; ++j) {
            const int mi = m0 + brow[j] - TN;
            if (mi >= g.m) continue;
            uint16_t* y = g.y + (int64_t)mi * g.ldy;
#pragma unroll
            for (int i = 0; i < FN; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int ni = nw + 32 * i + 8 * q;
                    if (vec && ni + 3 < g.n) {
                        *reinterpret_cast<u2*>(y + ni) = u2{narrow2(acc[i][j][4 * q], acc[i][j][4 * q + 1], g.kind),
                                                            narrow2(acc[i][j][4 * q + 2], acc[i][j][4 * q + 3], g.kind)};
                    } else {
#pragma unroll
                        for (int c = 0; c < 4; ++c)
                            if (ni + c < g.n) y[ni + c] = narrow(acc[i][j][4 * q + c], g.kind);
                    }
                }
        }
    } else {
#pragma unroll
        for (int j = 0; j < FM; ++j) {
            const int mi = m0 + brow[j] - TN;
            if (mi >= g.m) continue;
            const int xe = g.xe ? g.xe[mi] : 0;
            const int ge = OUT == OUT_GRAD && g.ge ? g.ge[mi] : 0;
#pragma unroll
            for (int i = 0; i < FN / 2; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int ni = nw + 32 * i + 8 * q;
                    float gv[4], uv[4];
                    int e0[4] = {0, 0, 0, 0}, e1[4] = {0, 0, 0, 0};
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        gv[c] = acc[i][j][4 * q + c];
                        uv[c] = acc[i + FN / 2][j][4 * q + c];
                        if (g.we0 && ni + c < g.n) { e0[c] = g.we0[ni + c]; e1[c] = g.we1[ni + c]; }
                        if (g.xe || g.we0) { gv[c] = ldexpf(gv[c], xe + e0[c]); uv[c] = ldexpf(uv[c], xe + e1[c]); }
                    }
                    if constexpr (OUT == OUT_GATED) {
                        uint16_t* y = g.y + (int64_t)mi * g.ldy;
#pragma unroll
                        for (int c = 0; c < 4; ++c) gv[c] = act_value(gv[c], g.act) * uv[c];
                        if (vec && ni + 3 < g.n) {
                            *reinterpret_cast<u2*>(y + ni) = u2{narrow2(gv[0], gv[1], g.kind), narrow2(gv[2], gv[3], g.kind)};
                        } else {
#pragma unroll
                            for (int c = 0; c < 4; ++c)
                                if (ni + c < g.n) y[ni + c] = narrow(gv[c], g.kind);
                        }
                    } else {
                        // columns n..np-1 are padding of the products that follow: zeros
                        const uint16_t* dh = g.dh + (int64_t)mi * g.ldh;
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            float dg = 0.f, du = 0.f;
                            if (ni + c < g.n) {
                                const float d = wide(dh[ni + c], g.kind);
                                float value, slope;
                                act_both(gv[c], g.act, value, slope);
                                dg = ldexpf(d * uv[c] * slope, e0[c] - ge);
                                du = ldexpf(d * value, e1[c] - ge);
                            }
                            gv[c] = dg;
                            uv[c] = du;
                        }
                        if (ni < g.np) {                        // np is a multiple of 64: whole groups of four
                            uint16_t* y = g.grad + (int64_t)mi * 2 * g.np + ni;
                            *reinterpret_cast<u2*>(y) = u2{narrow2(gv[0], gv[1], HALF), narrow2(gv[2], gv[3], HALF)};
                            *reinterpret_cast<u2*>(y + g.np) = u2{narrow2(uv[0], uv[1], HALF), narrow2(uv[2], uv[3], HALF)};
                        }
                    }
                }
        }
    }
}

template <int HALF, int TN, int TM, int WN, int WM, int OUT>
int launch(const Gemm& g, hipStream_t st) {
    constexpr int TNE = OUT == OUT_PLAIN ? TN : TN / 2;
    const int64_t nt = (g.n + TNE - 1) / TNE, mt = (g.m + TM - 1) / TM;
    if (nt * mt > INT32_MAX) return fail(SPA_ERR_ARG, "product: %d x %d outputs are too many", g.m, g.n);
    hipLaunchKernelGGL((k_gemm<HALF, TN, TM, WN, WM, OUT>), dim3((unsigned)(nt * mt)), dim3(WN * WM * 64), 0, st, g);
    SPA_HIP_TRY(hipGetLastError());
    return SPA_OK;
}

template <int HALF, int OUT>
int pick(const Gemm& g, hipStream_t st) {
    constexpr int D = OUT == OUT_PLAIN ? 1 : 2;
    const int64_t big = (int64_t)((g.n * D + 255) / 256) * ((g.m + 255) / 256);
    if (big >= 192) return launch<HALF, 256, 256, 2, 4, OUT>(g, st);
    if (g.m <= 64) return launch<HALF, 128, 64, 2, 2, OUT>(g, st);
    return launch<HALF, 128, 128, 2, 2, OUT>(g, st);
}

}  // namespace

int gemm(const Gemm& g, hipStream_t st) {
    if (g.half == SRC_BF16) {
        if (g.grad) return pick<SRC_BF16, OUT_GRAD>(g, st);
        return g.w1 ? pick<SRC_BF16, OUT_GATED>(g, st) : pick<SRC_BF16, OUT_PLAIN>(g, st);
    }
    if (g.grad) return pick<SRC_F16, OUT_GRAD>(g, st);
    return g.w1 ? pick<SRC_F16, OUT_GATED>(g, st) : pick<SRC_F16, OUT_PLAIN>(g, st);
}

}  // namespace lin
}  // namespace spa
