// The products for few input rows (up to FEW_ROWS): every weight is read once and used for all of them, so
// the weights' bytes are the floor. A workgroup of 8 waves computes 16 weight rows (16 of each matrix in the
// gated form) for all input rows; the waves share k and join their sums in LDS, in the order of the waves.
// One row of 12288 x 4096: BF16 19.1 us (5.3 TB/s, the memory's bound), IQ4_XS 33 us, bound by the decoding.
#include "../../include/seedpack_amd.h"
#include "few.h"
#include "launch.h"

namespace spa {
namespace lin {
namespace {

constexpr int WAVES = 8, KC = 1024, KW = KC / WAVES;          // k of a chunk, and each wave's part of it

// the input rows' fragments of one step of 32 k: row lane & 15 of tile j, k0 + 8 (lane / 16) ..
template <int MT>
__device__ __forceinline__ void load_x(const Few& f, int k0, u4 (&x)[MT]) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int j = 0; j < MT; ++j) {
        const int m = 16 * j + (lane & 15);
        x[j] = m < f.m ? *reinterpret_cast<const u4*>(f.x + (int64_t)m * f.ldx + k0 + 8 * (lane >> 4)) : u4{0, 0, 0, 0};
    }
}

template <int KIND>
__device__ __forceinline__ void halves(u4 raw, bf8& hi, bf8& lo) {                  // F16 values as two BF16 parts, exact
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = wide(raw[i] & 0xffffu, SRC_F16);
        v[2 * i + 1] = wide(raw[i] >> 16, SRC_F16);
    }
    split8(v, hi, lo);
}

// acc += x w for weights given as 8 floats a lane (weight row lane & 15, the k of load_x)
template <int KIND, int MT>
__device__ __forceinline__ void step(const u4 (&x)[MT], const float (&v)[8], f4 (&acc)[MT]) {
    bf8 wh, wl;
    split8(v, wh, wl);
#pragma unroll
    for (int j = 0; j < MT; ++j) {
        if (KIND == SRC_BF16) {
            const bf8 xb = __builtin_bit_cast(bf8, x[j]);
            acc[j] = mul_bf(xb, wl, acc[j]);
            acc[j] = mul_bf(xb, wh, acc[j]);
        } else {
            bf8 xh, xl;
            halves<KIND>(x[j], xh, xl);
            acc[j] = mul_bf(xh, wl, acc[j]);
            acc[j] = mul_bf(xl, wh, acc[j]);
            acc[j] = mul_bf(xh, wh, acc[j]);
        }
    }
}

struct Never {                                                   // of exact products: sums stay as they are
    static constexpr bool ANEW = false;
};

// Block types: a chunk of 1024 k of the 16 rows is copied to LDS as it lies (whole 16-byte words around each
// row's bytes), and each lane decodes 8 weights of its row in a step.
template <int T, int QK, int BS, int KIND, int MT, bool TWO>
__global__ __launch_bounds__(WAVES * 64) void k_few(const FewArgs a, DQ t) {
    const Few& f = a.f;
    constexpr int RB = KC / QK * BS, PITCH = (RB + 15 + 15) / 16 * 16 + 16, ROWS = 16 * (1 + TWO);
    constexpr int RED = WAVES * (1 + TWO) * MT * 256 * 4;
    constexpr int SIZE = ROWS * PITCH + 16 > RED ? ROWS * PITCH + 16 : RED;
    __shared__ __align__(16) uint8_t mem[SIZE];
    __shared__ int8_t kv[16];
    if (T == 20 || T == 23) {
        if (threadIdx.x < 16) kv[threadIdx.x] = KV_IQ4NL[threadIdx.x];
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n0 = blockIdx.x * 16;
    const int row = lane & 15, kl = 8 * (lane >> 4);
    f4 acc[1 + TWO][MT];
#pragma unroll
    for (int s = 0; s <= TWO; ++s)
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[s][j] = f4{0, 0, 0, 0};

    for (int c0 = 0; c0 < f.k; c0 += KC) {
        const int kn = tmin(KC, f.k - c0), bytes = kn / QK * BS;
        const int64_t at = (int64_t)(c0 / QK) * BS;
        constexpr int WORDS = PITCH / 16 - 1;
        __syncthreads();
        for (int i = threadIdx.x; i < ROWS * WORDS; i += WAVES * 64) {
            const int r = i / WORDS, u = i - r * WORDS, n = tmin(n0 + (r & 15), f.n - 1);
            const uint8_t* w = TWO && r >= 16 ? f.w1 : f.w0;
            const uint8_t* src = w + n * a.rowbytes + at;
            const uint8_t* p = reinterpret_cast<const uint8_t*>(reinterpret_cast<uintptr_t>(src) & ~(uintptr_t)15) + 16 * u;
            if (p >= src + bytes) continue;
            u4* d = reinterpret_cast<u4*>(mem + r * PITCH + 16 * u);
            if (p >= w && p + 16 <= w + f.wbytes) {
                *d = *reinterpret_cast<const u4*>(p);
            } else {                                              // the matrix's first or last word: its own bytes only
                uint8_t* b = reinterpret_cast<uint8_t*>(d);
                for (int k = 0; k < 16; ++k)
                    if (p + k >= w && p + k < w + f.wbytes) b[k] = p[k];
            }
        }
        __syncthreads();
#pragma unroll 2
        for (int s = 0; s < KW / 32; ++s) {
            const int k = wave * KW + 32 * s;
            if (k >= kn) break;
            u4 x[MT];
            load_x<MT>(f, c0 + k, x);
            const int e = k + kl, blk = e / QK;
#pragma unroll
            for (int h = 0; h <= TWO; ++h) {
                const uint8_t* src = (h ? f.w1 : f.w0) + (int64_t)tmin(n0 + row, f.n - 1) * a.rowbytes + at;
                const FastBlk b{{mem, (row + 16 * h) * PITCH + (int)(reinterpret_cast<uintptr_t>(src) & 15) + blk * BS}};
                float v[8], q[4];
                dq4<T>(b, e - blk * QK, t, kv, q);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = q[i];
                dq4<T>(b, e - blk * QK + 4, t, kv, q);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[4 + i] = q[i];
                step<KIND, MT>(x, v, acc[h]);
            }
        }
    }
    finish<WAVES, MT, TWO, false>(f, n0, reinterpret_cast<float*>(mem), acc, Direct<T, QK, BS>{a, t, kv});
}

// 16-bit weights: fragments straight from memory, the loads of four steps under way at once. LINED: rows of whole
// steps at 16-byte addresses. WORDS: rows that begin at words. ANYWHERE: at any number (three rows of 14221 x 8471: 95 us
// with 16-byte loads from there, 59 by whole words; 3649 x 10174, whose rows begin at words, 20 and 22). The step that
// reaches past a row's end is read number by number, with zeros (the inputs hold zeros there too, but the next
// row's weights may be infinite).
enum Lie { ANYWHERE, WORDS, LINED };
template <int WKIND, int KIND, int MT, bool TWO, Lie LIE, int W>
__global__ __launch_bounds__(W * 64) void k_few16(const FewArgs a) {
    const Few& f = a.f;
    __shared__ float red[W * (1 + TWO) * MT * 256];
    constexpr int U = MT > 2 ? 2 : 4, STEP = W * 32;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n0 = blockIdx.x * 16;
    const int kl = 8 * (lane >> 4), cols = (int)(a.rowbytes / 2);
    const int64_t wrow = (int64_t)tmin(n0 + (lane & 15), f.n - 1) * a.rowbytes;
    f4 acc[1 + TWO][MT];
#pragma unroll
    for (int s = 0; s <= TWO; ++s)
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[s][j] = f4{0, 0, 0, 0};
    for (int k0 = wave * 32; k0 < f.k; k0 += U * STEP) {
        u4 x[U][MT], w[U][1 + TWO];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = k0 + u * STEP;
            if (k >= f.k) break;
            if constexpr (MT == 1) {
                load_x<MT>(f, k, x[u]);
            } else {                                              // as fragments
#pragma unroll
                for (int j = 0; j < MT; ++j) x[u][j] = reinterpret_cast<const u4*>(f.x)[(k / 32 * MT + j) * 64 + lane];
            }
#pragma unroll
            for (int h = 0; h <= TWO; ++h) {
                const uint8_t* p = (h ? f.w1 : f.w0) + wrow + 2 * (k + kl);
                if (LIE == LINED) {
                    w[u][h] = *reinterpret_cast<const u4*>(p);
                } else if (k + 32 <= cols) {
                    if (LIE == WORDS) __builtin_memcpy(&w[u][h], p, 16);
                    else w[u][h] = load8_words(reinterpret_cast<const uint16_t*>(p));
                } else {
                    const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t lo = k + kl + 2 * i < cols ? q[2 * i] : 0, hi = k + kl + 2 * i + 1 < cols ? q[2 * i + 1] : 0;
                        w[u][h][i] = lo | (hi << 16);
                    }
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (k0 + u * STEP >= f.k) break;
#pragma unroll
            for (int h = 0; h <= TWO; ++h) {
                if (WKIND == KIND) {
#pragma unroll
                    for (int j = 0; j < MT; ++j) acc[h][j] = mul16<KIND>(x[u][j], w[u][h], acc[h][j]);
                } else {
                    float v[8];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        v[2 * i] = wide(w[u][h][i] & 0xffffu, WKIND);
                        v[2 * i + 1] = wide(w[u][h][i] >> 16, WKIND);
                    }
                    step<KIND, MT>(x[u], v, acc[h]);
                }
            }
        }
    }
    if constexpr (WKIND == KIND) finish<W, MT, TWO, false>(f, n0, red, acc, Never());
    else finish<W, MT, TWO, false>(f, n0, red, acc, Direct<WKIND == SRC_F16 ? 1 : 30, 1, 2>{a, DQ{nullptr}, nullptr});
}

template <int T, int QK, int BS, int KIND, bool TWO>
int launch(const FewArgs& given, DQ t, uint16_t* frags, hipStream_t st) {
    const dim3 grid((unsigned)((given.f.n + 15) / 16)), block(WAVES * 64);
    if constexpr (T == 1 || T == 30) {
        constexpr int WK = T == 1 ? SRC_F16 : SRC_BF16;
        FewArgs a = given;
        const int tiles = few_tiles(T, a.f.m);
        if (tiles > 1) {
            const int rc = fragments(a.f, Frags{frags, tiles, a.f.k, false}, st);
            if (rc) return rc;
            a.f.x = frags;
        }
        const bool lined = a.rowbytes == 2 * (int64_t)a.f.k && ((reinterpret_cast<uintptr_t>(a.f.w0) | reinterpret_cast<uintptr_t>(a.f.w1)) & 15) == 0;
        const bool words = a.rowbytes % 4 == 0;                   // 16-bit matrices begin at 16-byte addresses
        // Few weight rows fill the device with waves only if more of them share a row's k (one row of 4060 x 5795
        // with 8 waves: 80 us), and a long k keeps 16 busy whatever the rows: one row with 8 and with 16 waves, us:
        //     k      n = 4096       8192      12288       32768
        //  1024     6.1  6.1     6.1  6.1    7.3  8.2   13.4 16.9
        //  2048     7.4  6.7    11.2  9.0   14.9 12.0   31.0 25.1
        //  4096     9.9  9.6    17.1 15.3   23.3 21.0   52.9 49.0
        //  8192    19.0 18.7    32.3 30.8   45.2 43.1  108.3 99.1
#define SPA_FEW16(MT, W)                                                                                    \
    do {                                                                                                    \
        if (lined) hipLaunchKernelGGL((k_few16<WK, KIND, MT, TWO, LINED, W>), grid, dim3(W * 64), 0, st, a);         \
        else if (words) hipLaunchKernelGGL((k_few16<WK, KIND, MT, TWO, WORDS, W>), grid, dim3(W * 64), 0, st, a);    \
        else hipLaunchKernelGGL((k_few16<WK, KIND, MT, TWO, ANYWHERE, W>), grid, dim3(W * 64), 0, st, a);            \
    } while (0)
        if (a.f.m <= 16) {
            if (a.f.n < 8192 || a.f.k >= 2048) SPA_FEW16(1, 16);
            else SPA_FEW16(1, 8);
        } else if (a.f.m <= 32) {
            SPA_FEW16(2, 8);
        } else {
            SPA_FEW16(4, 8);
        }
#undef SPA_FEW16
    } else {
        if (given.f.m <= 16) hipLaunchKernelGGL((k_few<T, QK, BS, KIND, 1, TWO>), grid, block, 0, st, given, t);
        else if (given.f.m <= 32) hipLaunchKernelGGL((k_few<T, QK, BS, KIND, 2, TWO>), grid, block, 0, st, given, t);
        else hipLaunchKernelGGL((k_few<T, QK, BS, KIND, 4, TWO>), grid, block, 0, st, given, t);
    }
    SPA_HIP_TRY(hipGetLastError());
    return SPA_OK;
}

template <int T, int QK, int BS>
int pick(const FewArgs& a, DQ t, uint16_t* frags, hipStream_t st) {
    if (a.f.w1) return a.f.kind == SRC_BF16 ? launch<T, QK, BS, SRC_BF16, true>(a, t, frags, st) : launch<T, QK, BS, SRC_F16, true>(a, t, frags, st);
    return a.f.kind == SRC_BF16 ? launch<T, QK, BS, SRC_BF16, false>(a, t, frags, st) : launch<T, QK, BS, SRC_F16, false>(a, t, frags, st);
}

}  // namespace

int few(const Few& f, uint16_t* frags, hipStream_t st) {
    DQ t{nullptr};
    const int ti = iq_table_index(f.type);
    if (ti >= 0) {
        IqDeviceTable tab;
        const int rc = iq_device_table(ti, &tab, st);
        if (rc) return rc;
        t.grid = tab.grid;
    }
    if (coded(f.type)) return few_codes(f, frags, st);
    FewArgs a{f, 0, f.x};
    switch (f.type) {
#define SPA_FEW(T, QK, BS)                                 \
    case T:                                                \
        a.rowbytes = f.rowbytes;                           \
        return pick<T, QK, BS>(a, t, frags, st);
        SPA_FEW(1, 1, 2) SPA_FEW(30, 1, 2)
        SPA_FEW(3, 32, 20) SPA_FEW(6, 32, 22) SPA_FEW(7, 32, 24)
        SPA_FEW(10, 256, 84) SPA_FEW(11, 256, 110)
        SPA_FEW(16, 256, 66) SPA_FEW(17, 256, 74) SPA_FEW(18, 256, 98) SPA_FEW(19, 256, 50) SPA_FEW(20, 32, 18)
        SPA_FEW(21, 256, 110) SPA_FEW(22, 256, 82) SPA_FEW(23, 256, 136) SPA_FEW(29, 256, 56) SPA_FEW(42, 64, 18)
#undef SPA_FEW
        default: return fail(SPA_ERR_TYPE, "weights of type %d are not supported", f.type);
    }
}

}  // namespace lin
}  // namespace spa
