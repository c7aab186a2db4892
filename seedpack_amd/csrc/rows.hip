// The passes over rows around the products of gemm.hip: operands brought into the form that it takes
// (padded, converted, transposed), the powers of two that conversions take out, and the adapters' first
// product. All but the decoding of blocks and the adapters' products are bound by memory or a launch's latency.
#include "../../include/seedpack_amd.h"
#include "dq.h"
#include "launch.h"
#include "linear.h"

namespace spa {
namespace lin {
namespace {

// eight elements from k on, zeros from n on. The address may be any element's: gfx950 loads 16 bytes from any byte.
// WORDS false: see load8_words
template <bool WORDS = true>
__device__ __forceinline__ void load8(const uint16_t* row, int64_t k, int64_t n, u4& v) {
    if (k + 8 <= n) {
        if (WORDS) __builtin_memcpy(&v, row + k, 16);
        else v = load8_words(row + k);
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t a = k + 2 * i < n ? row[k + 2 * i] : 0, b = k + 2 * i + 1 < n ? row[k + 2 * i + 1] : 0;
        v[i] = a | (b << 16);
    }
}

__global__ __launch_bounds__(256) void k_pack(const uint16_t* __restrict__ src, int64_t ld, int64_t rows, int64_t k,
                                              uint16_t* __restrict__ dst, int64_t kp) {
    const int64_t per = kp / 8, total = rows * per;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
        const int64_t r = i / per, c = (i - r * per) * 8;
        u4 h;
        load8(src + r * ld, c, k, h);
        *reinterpret_cast<u4*>(dst + r * kp + c) = h;
    }
}

// a workgroup's largest or total float, the same in every lane; in an order of its own shape only
template <bool MAX, int LANES = 256>
__device__ __forceinline__ float reduce(float v, float* lds) {
#pragma unroll
    for (int s = 32; s; s >>= 1) {
        const float o = __shfl_xor(v, s);
        v = MAX ? fmaxf(v, o) : v + o;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lds[0];
#pragma unroll
    for (int w = 1; w < LANES / 64; ++w) v = MAX ? fmaxf(v, lds[w]) : v + lds[w];
    return v;
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
// A row of up to KEEP numbers a lane stays in registers between the search for its largest and its conversion;
// KEEP = 0: any row, read twice. 2053 x 12288: 23 us, 4.4 TB/s read and written.
template <int KEEP, int LANES>
__global__ __launch_bounds__(LANES) void k_half_rows(const uint16_t* __restrict__ src, int kind, int64_t ld, int64_t k,
                                                   uint16_t* __restrict__ dst, int64_t kp, int64_t ldd, int32_t* __restrict__ e_out,
                                                   float* __restrict__ norm, bool twice) {
    __shared__ float lds[LANES / 64];
    const int64_t row = blockIdx.x;
    src += row * ld;
    dst += row * ldd;
    float most = 0.f;
    u4 held[KEEP ? KEEP / 8 : 1];
    auto largest = [&](const u4& h) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            most = fmaxf(most, fmaxf(size_of(wide(h[i] & 0xffffu, kind)), size_of(wide(h[i] >> 16, kind))));
    };
    if constexpr (KEEP != 0) {
#pragma unroll
        for (int t = 0; t < KEEP / 8; ++t) {
            const int64_t c = t * (8 * LANES) + threadIdx.x * 8;
            held[t] = u4{0, 0, 0, 0};
            if (c < k) load8(src, c, k, held[t]);
        }
#pragma unroll
        for (int t = 0; t < KEEP / 8; ++t) largest(held[t]);
    } else {
        for (int64_t c = threadIdx.x * 8; c < k; c += 8 * LANES) {
            u4 h;
            load8(src, c, k, h);
            largest(h);
        }
    }
    const int e = exponent_for(reduce<true, LANES>(most, lds));
    float sum = 0.f;
    auto convert = [&](int64_t c, u4 h) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a = ldexpf(wide(h[i] & 0xffffu, kind), -e), b = ldexpf(wide(h[i] >> 16, kind), -e);
            sum = fmaf(size_of(a), size_of(a), fmaf(size_of(b), size_of(b), sum));
            h[i] = narrow2(a, b, SRC_F16);
        }
        *reinterpret_cast<u4*>(dst + c) = h;
        if (twice) *reinterpret_cast<u4*>(dst + kp + c) = u4{finite2(h[0]), finite2(h[1]), finite2(h[2]), finite2(h[3])};
    };
    if constexpr (KEEP != 0) {
#pragma unroll
        for (int t = 0; t < KEEP / 8; ++t) {
            const int64_t c = t * (8 * LANES) + threadIdx.x * 8;
            if (c < kp) convert(c, held[t]);
        }
    } else {
        for (int64_t c = threadIdx.x * 8; c < kp; c += 8 * LANES) {
            u4 h;
            load8(src, c, k, h);
            convert(c, h);
        }
    }
    if (threadIdx.x == 0) e_out[row] = e;
    if (norm) {
        sum = reduce<false, LANES>(sum, lds);
        if (threadIdx.x == 0) norm[row] = fminf(ldexpf(sqrtf(sum), e), 3e38f);
    }
}

typedef uint16_t h2u __attribute__((ext_vector_type(2)));

// what a block's weights are at most in size, by its header: scale (and offset) times the largest code
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

// A row's blocks go to LDS, TILE weights at a time; a row of one tile is there before its headers are looked at, so
// that its bytes are waited for once. Longer rows: the headers from memory first. FULL: with the norm or the rest.
// A quantizer's largest weight of a row lies within 2^1.4 of its headers' bound (19 types, normal weights), but where
// codes are small or zero the bound may be any power of two above: a row whose largest weight turns out 2^5 or more below
// is converted once more by that weight, so that weights are there to 2^-34 of their row's largest. The look at the
// halves as they leave costs 1.2 us of 16 for Q4_K 4096 x 4096. (Decoded once into registers and converted by the true
// largest: 300 rows beside Q6_K 4096 x 8192 in all 78 us, 68 this way.)
// Bound by the decoding's instructions: 33 us for Q4_K 4096 x 12288 (27 instructions a weight with four weights a
// lane and the norm always summed: 44 us), 3.9 TB/s read and written.
template <int T, int QK, int BS, int TILE, bool FULL>
__global__ __launch_bounds__(256) void k_half_blocks(const uint8_t* __restrict__ src, int64_t k, uint16_t* __restrict__ dst,
                                                     int64_t kp, int64_t ldd, int32_t* __restrict__ e_out, float* __restrict__ norm, bool rest,
                                                     DQ t, int align) {
    constexpr int TB = TILE / QK, TBYTES = TB * BS;
    __shared__ __align__(16) uint8_t tile[TBYTES + 16];
    __shared__ int8_t kv[16];
    __shared__ float lds[4];
    __shared__ int near;
    if (threadIdx.x == 0) near = 0;
    if (T == 20 || T == 23) {
        if (threadIdx.x < 16) kv[threadIdx.x] = KV_IQ4NL[threadIdx.x];
    }
    const int64_t row = blockIdx.x, nb = k / QK;
    src += row * nb * BS;
    dst += row * ldd;
    auto stage = [&](int64_t b0, int n) {
        const int bytes = n * BS;
        const uint8_t* s = src + b0 * BS;
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
    };
    const bool one = nb <= TB;
    if (one) stage(0, (int)nb);
    float most = 0.f;
    for (int64_t b = threadIdx.x; b < nb; b += 256) most = fmaxf(most, block_bound<T>((one ? tile : src) + b * BS));
    // f(the first of eight weights, all eight): what a block's header says of them is worked out once
    auto each = [&](auto f) {
        for (int64_t b0 = 0; b0 < nb; b0 += TB) {
            const int n = (int)(nb - b0 < TB ? nb - b0 : TB);
            if (!one) {
                __syncthreads();
                stage(b0, n);
            }
            for (int q = threadIdx.x; q < n * (QK / 8); q += 256) {
                const int o = q * 8, blk = o / QK;
                const FastBlk in{{tile, blk * BS}};
                float v[8], w[4];
                dq4<T>(in, o - blk * QK, t, kv, w);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = w[i];
                dq4<T>(in, o - blk * QK + 4, t, kv, w);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[4 + i] = w[i];
                f(b0 * QK + o, v);
            }
        }
    };
    const float bound = reduce<true>(most, lds);
    int e = exponent_for(bound);
    float sum;
    for (bool first = true;; first = false) {
        h2u top = {0, 0};                                         // the largest halves, without their signs
        sum = 0.f;
        each([&](int64_t at, float (&v)[8]) {
            u4 h;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = ldexpf(v[i], -e);
            if (FULL && norm) {
#pragma unroll
                for (int i = 0; i < 8; ++i) sum = fmaf(size_of(v[i]), size_of(v[i]), sum);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                h[i] = narrow2(v[2 * i], v[2 * i + 1], SRC_F16);
                const uint32_t size = h[i] & 0x7fff7fffu;
                top = __builtin_elementwise_max(top, __builtin_bit_cast(h2u, size));
            }
            *reinterpret_cast<u4*>(dst + at) = h;
            if (FULL && rest) {                                   // what binary16 leaves over (nothing of infinities)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float r = wide((h[i >> 1] >> (16 * (i & 1))) & 0xffffu, SRC_F16);
                    v[i] = size_of(r) == fabsf(r) ? v[i] - r : 0.f;
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) h[i] = narrow2(v[2 * i], v[2 * i + 1], SRC_F16);
                *reinterpret_cast<u4*>(dst + kp + at) = h;
            }
        });
        if (!first) break;
        const uint32_t mine = tmax(top[0], top[1]);
        if (__ballot(mine >= 0x6400u && mine < 0x7c00u)) near = 1;   // 2^10 and above: the same from every writer
        __syncthreads();
        if (near || !(bound > 0.f)) break;
        const uint32_t bits = (uint32_t)reduce<true>((float)mine, lds);
        most = wide(bits, SRC_F16);
        if (bits == 0 || bits >= 0x7c00u) {                       // nothing left, or infinities: by the numbers themselves
            most = 0.f;
            each([&](int64_t, float (&v)[8]) {
#pragma unroll
                for (int i = 0; i < 8; ++i) most = fmaxf(most, ldexpf(size_of(v[i]), -e));
            });
            most = reduce<true>(most, lds);
        }
        const int over = most > 0.f ? -exponent_for(most) : 0;
        if (over < 5) break;
        e -= over;
    }
    for (int64_t c = k + threadIdx.x; c < kp; c += 256) {
        dst[c] = 0;
        if (FULL && rest) dst[kp + c] = 0;
    }
    if (threadIdx.x == 0) e_out[row] = e;
    if (FULL && norm) {
        sum = reduce<false>(sum, lds);
        if (threadIdx.x == 0) norm[row] = fminf(ldexpf(sqrtf(sum), e), 3e38f);
    }
}

// 2-norms of the rows of three F16 matrices of k columns, a workgroup a row: x's, then those of both
// weights. 4096 and 2 x 12288 rows of 4096: 47 us, 5.0 TB/s.
struct Norms {
    const uint16_t *x, *w0, *w1;
    int64_t ldx, m, n, k;
    float *xn, *n0, *n1;
};
__global__ __launch_bounds__(256) void k_norms(const Norms q) {
    __shared__ float lds[4];
    const int64_t row = blockIdx.x, at = row < q.m ? row : (row - q.m) % q.n;
    const bool first = row - q.m < q.n;
    const uint16_t* src = row < q.m ? q.x + at * q.ldx : (first ? q.w0 : q.w1) + at * q.k;
    float sum = 0.f;
    for (int64_t c = threadIdx.x * 8; c < q.k; c += 2048) {
        u4 h;
        load8(src, c, q.k, h);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a = size_of(wide(h[i] & 0xffffu, SRC_F16)), b = size_of(wide(h[i] >> 16, SRC_F16));
            sum = fmaf(a, a, fmaf(b, b, sum));
        }
    }
    sum = reduce<false>(sum, lds);
    if (threadIdx.x == 0) (row < q.m ? q.xn : (first ? q.n0 : q.n1))[at] = sqrtf(sum);
}

// 64 x 64 tiles through LDS: read along a row's columns, written along a column's rows, eight numbers a lane both
// ways. 12288 x 4096: 35 us, 5.7 TB/s read and written. SCALED: F16 rows of src have 2^re taken out, rows of dst
// get 2^ce taken out in its place (4096 x 24576: 60 us without, 87 with).
template <bool SCALED>
__global__ __launch_bounds__(256) void k_transpose(const uint16_t* __restrict__ src, int64_t ld, int64_t rows, int64_t cols,
                                                   uint16_t* __restrict__ dst, int64_t ldd, int64_t rp, int64_t tiles_c,
                                                   const int32_t* __restrict__ re, const int32_t* __restrict__ ce) {
    __shared__ uint16_t t[64][66];                                // 33 words a row: a column's reads meet few banks twice
    const int64_t r0 = blockIdx.x / tiles_c * 64, c0 = blockIdx.x % tiles_c * 64;
    int out[8];                                                   // of the lane's eight columns, which both its loads are of
    if constexpr (SCALED) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int64_t C = c0 + (threadIdx.x & 7) * 8 + k;
            out[k] = ce[C < cols ? C : cols - 1];
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int u = i * 256 + threadIdx.x, r = u >> 3, c = (u & 7) * 8;
        const int64_t R = r0 + r, C = c0 + c;
        u4 v = {0, 0, 0, 0};
        if (R < rows && C < cols) {
            load8(src + R * ld, C, cols, v);
            if constexpr (SCALED) {
                const int e = re[R];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const uint16_t h = (uint16_t)(v[k >> 1] >> (16 * (k & 1)));
                    const uint32_t s = narrow(ldexpf(wide(h, SRC_F16), e - out[k]), SRC_F16);
                    v[k >> 1] = k & 1 ? (v[k >> 1] & 0xffffu) | s << 16 : (v[k >> 1] & 0xffff0000u) | s;
                }
            }
        }
        uint32_t* p = reinterpret_cast<uint32_t*>(&t[r][c]);
#pragma unroll
        for (int k = 0; k < 4; ++k) p[k] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int u = i * 256 + threadIdx.x, c = u >> 3, r = (u & 7) * 8;
        const int64_t R = r0 + r, C = c0 + c;
        if (C < cols && R < rp) {                                 // rp and ldd are multiples of 8, dst 16-byte aligned
            u4 v;
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = (uint32_t)t[r + 2 * k][c] | ((uint32_t)t[r + 2 * k + 1][c] << 16);
            *reinterpret_cast<u4*>(dst + C * ldd + R) = v;
        }
    }
}

// The largest 2-norm and the largest power of two of both matrices' rows, by one workgroup: 6 us for 12288.
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
// 1000 rows of 12288: 9 us.
__global__ __launch_bounds__(256) void k_grad_exponents(const uint16_t* __restrict__ dh, int kind, int64_t ld, int64_t n,
                                                        const float* __restrict__ xnorm, const Top* __restrict__ top,
                                                        int32_t* __restrict__ e) {
    __shared__ float lds[4];
    const int64_t row = blockIdx.x;
    float most = 0.f;
    for (int64_t c = threadIdx.x * 8; c < n; c += 2048) {
        u4 h;
        load8(dh + row * ld, c, n, h);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            most = fmaxf(most, fmaxf(size_of(wide(h[i] & 0xffffu, kind)), size_of(wide(h[i] >> 16, kind))));
    }
    most = reduce<true>(most, lds);
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

// The same bounds for F16 weights beside F16 inputs, of each row of the inner gradients (for dx) and of each column
// (for the weights' gradients, sums over rows): the largest |dh| |w_n| of a row, the largest |dh| |x_m| of a column. One
// pass over dh, 512 columns and a run of rows a workgroup, its waves every fourth row: 47 us for 4096 x 12288 (2.1 TB/s),
// 5.6 of joining; 517 x 2053, whose rows begin at any number, 7.6 and 4.4.
constexpr int TOP_COLS = 512, TOP_RUN = 16, TOP_PIECES = 64;
struct Tops {
    const uint16_t* dh;
    int64_t ld, m, n, np, run;
    const float *xn, *n0, *n1;
    float *rows, *cols;       // [column tile][m], [run][np]
    int pieces, tiles;
    int32_t *ge, *ce;
};
template <bool WORDS>
__global__ __launch_bounds__(256) void k_tops(const Tops q) {
    __shared__ float lds[3][TOP_COLS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t c = (int64_t)blockIdx.x * TOP_COLS + 8 * lane, r0 = blockIdx.y * q.run, r1 = r0 + q.run < q.m ? r0 + q.run : q.m;
    float top[8] = {0, 0, 0, 0, 0, 0, 0, 0}, w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = c + i < q.n ? fmaxf(q.n0[c + i], q.n1[c + i]) : 0.f;
    for (int64_t at = r0 + wave; at < r1; at += 16) {             // four rows' loads under way at once
        u4 h[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            h[u] = u4{0, 0, 0, 0};
            if (at + 4 * u < r1 && c < q.n) load8<WORDS>(q.dh + (at + 4 * u) * q.ld, c, q.n, h[u]);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t r = at + 4 * u;
            const float a = q.xn[r < r1 ? r : r1 - 1];
            float row = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float d = size_of(wide((h[u][i >> 1] >> (16 * (i & 1))) & 0xffffu, SRC_F16));
                top[i] = fmaxf(top[i], a * d);
                row = fmaxf(row, w[i] * d);
            }
#pragma unroll
            for (int s = 32; s; s >>= 1) row = fmaxf(row, __shfl_xor(row, s));
            if (lane == 0 && r < r1) q.rows[blockIdx.x * q.m + r] = row;
        }
    }
    if (wave) {
#pragma unroll
        for (int i = 0; i < 8; ++i) lds[wave - 1][i * 64 + lane] = top[i];
    }
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float v = fmaxf(fmaxf(top[i], lds[0][i * 64 + lane]), fmaxf(lds[1][i * 64 + lane], lds[2][i * 64 + lane]));
        if (c + i < q.np) q.cols[blockIdx.y * q.np + c + i] = v;
    }
}
__device__ __forceinline__ int bound_exponent(float a, float b) {
    int ea = 0, eb = 0;
    frexpf(a, &ea);
    frexpf(b, &eb);
    return a > 0.f && b > 0.f ? ea + eb + 1 - 15 : 0;
}
// dG' of column n goes with the up projection's norm, dU' with the gate's
__global__ __launch_bounds__(256) void k_exponents(const Tops q) {
    const int64_t i = blockIdx.x * 256ll + threadIdx.x;
    float v = 0.f;
    if (i < q.m) {
#pragma unroll 8
        for (int p = 0; p < q.tiles; ++p) v = fmaxf(v, q.rows[p * q.m + i]);
        q.ge[i] = bound_exponent(v, q.xn[i]);
    } else if (i < q.m + q.np) {
        const int64_t n = i - q.m;
#pragma unroll 8
        for (int p = 0; p < q.pieces; ++p) v = fmaxf(v, q.cols[p * q.np + n]);
        q.ce[n] = bound_exponent(v, n < q.n ? q.n1[n] : 0.f);
        q.ce[q.np + n] = bound_exponent(v, n < q.n ? q.n0[n] : 0.f);
    }
}

__global__ void k_zero_rows(uint16_t* p, int64_t ld, int64_t rows, int64_t k) {
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < rows * k; i += gridDim.x * 256ll) p[i / k * ld + i % k] = 0;
}

// low[m][r] = s_a sum_k x[m][k] A_a[r][k] for 16 MT rows a workgroup and one adapter: `most` workgroups take
// the adapters among the rows in turn, in rising order, most of them finding none. The whole tile is
// multiplied by the adapter's matrix and its own rows are kept. The 16 waves take 64 k (a line of each row)
// in turn, the loads of 128 or 256 k under way at once; up to 64 ranks at a time, so that x is read once for the
// usual ranks. Bound by the latency of its few workgroups' loads: 7 us for a row of 4096 at rank 16, 12 us for 32 rows
// with 16 adapters.
constexpr int LOW_WAVES = 16;
template <int KIND, int MT, int TILES, bool WORDS>
__global__ __launch_bounds__(LOW_WAVES * 64) void k_low(const uint16_t* __restrict__ x, int64_t ldx, int64_t m, int64_t k,
                                                        const uint16_t* __restrict__ a_all, const float* __restrict__ scale,
                                                        const int32_t* __restrict__ which, int pool, int rank,
                                                        float* __restrict__ low, int rp, int most, const Frags fr) {
    if (blockIdx.y >= (unsigned)most) {                           // the other job of the launch
        const int count = fr.tiles * (fr.k / 32) * 64, step = (gridDim.y - most) * gridDim.x * (LOW_WAVES * 64);
        for (int i = ((blockIdx.y - most) * gridDim.x + blockIdx.x) * (LOW_WAVES * 64) + threadIdx.x; i < count; i += step) fragment(fr, x, ldx, m, i);
        return;
    }
    __shared__ float part[LOW_WAVES][TILES][256];
    __shared__ int ids[16 * MT];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t m0 = (int64_t)blockIdx.x * 16 * MT;
    const int row = lane & 15, kc = (lane >> 4) * 8;
    int mine[MT];
    const uint16_t* xr[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int64_t mi = m0 + 16 * t + row;
        mine[t] = mi < m ? which[mi] : -1;
        xr[t] = x + (mi < m ? mi : m - 1) * ldx;
    }
    for (int i = threadIdx.x; i < 16 * MT; i += LOW_WAVES * 64) ids[i] = m0 + i < m ? which[m0 + i] : -1;
    if (blockIdx.y == 0) {                                        // rows without an adapter: zeros
        for (int i = threadIdx.x; i < 16 * MT * rp; i += LOW_WAVES * 64) {
            const int64_t mi = m0 + i / rp;
            if (mi < m) {
                const int a = which[mi];
                if (a < 0 || a >= pool) low[mi * rp + i % rp] = 0.f;
            }
        }
    }
    int a = -1;
    for (unsigned turn = 0;; ++turn) {                            // the same in every lane and wave
        int best = INT32_MAX;
#pragma unroll
        for (int t = 0; t < MT; ++t)
            if (mine[t] > a && mine[t] < pool) best = tmin(best, mine[t]);
#pragma unroll
        for (int s = 8; s; s >>= 1) best = tmin(best, __shfl_xor(best, s));
        a = __builtin_amdgcn_readfirstlane(best);
        if (a == INT32_MAX) return;
        if (turn == blockIdx.y) break;
    }
    const int64_t lines = (k + 63) / 64, turned = (int64_t)blockIdx.x * 5 % lines;
    const uint16_t* aa = a_all + (int64_t)a * rank * k;
    const float sa = scale[a];
    for (int r0 = 0; r0 < rp; r0 += 16 * TILES) {
        const int tiles = tmin(TILES, (rp - r0) / 16);
        const uint16_t* ar[TILES];
        f4 acc[MT][TILES];
#pragma unroll
        for (int j = 0; j < TILES; ++j) {
            const int r = r0 + 16 * j + row;                      // ranks beyond the last take its row: they are not kept
            ar[j] = aa + (int64_t)(r < rank ? r : rank - 1) * k;
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[t][j] = f4{0, 0, 0, 0};
        }
        constexpr int U = (TILES == 1 ? 8 : 4) / MT;              // steps of 32 k at once
        for (int64_t l = wave; l < lines; l += LOW_WAVES * (U / 2)) {
            u4 xv[U][MT], av[U][TILES];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                // workgroups begin at different lines: rows of a power of two apart lie in few memory channels
                const int64_t i = l + LOW_WAVES * (u / 2), at = i + turned < lines ? i + turned : i + turned - lines;
                const int64_t k0 = at * 64 + 32 * (u % 2) + kc;
                const bool in = i < lines && k0 < k;
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    xv[u][t] = u4{0, 0, 0, 0};
                    if (in) load8<WORDS>(xr[t], k0, k, xv[u][t]);
                }
#pragma unroll
                for (int j = 0; j < TILES; ++j) {
                    av[u][j] = u4{0, 0, 0, 0};
                    if (in && j < tiles) load8<WORDS>(ar[j], k0, k, av[u][j]);
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int j = 0; j < TILES; ++j) {
                    if (j >= tiles) break;
#pragma unroll
                    for (int t = 0; t < MT; ++t) {
                        if (KIND == SRC_BF16)
                            acc[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, xv[u][t]), __builtin_bit_cast(bf8, av[u][j]), acc[t][j], 0, 0, 0);
                        else
                            acc[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(hf8, xv[u][t]), __builtin_bit_cast(hf8, av[u][j]), acc[t][j], 0, 0, 0);
                    }
                }
        }
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < TILES; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c) part[wave][j][(4 * (lane >> 4) + c) * 16 + row] = acc[t][j][c];
            __syncthreads();
            const int i = threadIdx.x, j = i >> 8, mr = (i >> 4) & 15, r = r0 + 16 * j + (i & 15);
            const int64_t mi = m0 + 16 * t + mr;
            if (j < TILES && mi < m && r < rp && ids[16 * t + mr] == a) {
                float v = 0.f;
#pragma unroll
                for (int w = 0; w < LOW_WAVES; ++w) v += part[w][j][i & 255];
                low[mi * rp + r] = r < rank ? sa * v : 0.f;
            }
        }
    }
}

// the row's own adapter out of the products with all of them: part [piece][m][pool rank], AT pieces' loads under way
// at once
__global__ __launch_bounds__(256) void k_low_pick(const float* __restrict__ part, int pieces, const float* __restrict__ scale,
                                                  const int32_t* __restrict__ which, int64_t m, int pool, int rank, float* __restrict__ low,
                                                  int rp) {
    constexpr int AT = 8;
    const int64_t width = (int64_t)pool * rank, size = m * width;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < m * rp; i += gridDim.x * 256ll) {
        const int64_t mi = i / rp;
        const int r = (int)(i - mi * rp), a = which[mi];
        float v = 0.f;
        if (r < rank && a >= 0 && a < pool) {
            const float* p = part + mi * width + (int64_t)a * rank + r;
            for (int j = 0; j < pieces; j += AT) {
                float t[AT];
#pragma unroll
                for (int c = 0; c < AT; ++c) t[c] = p[tmin(j + c, pieces - 1) * size];     // those beyond the last are dropped
#pragma unroll
                for (int c = 0; c < AT; ++c)
                    if (j + c < pieces) v += t[c];
            }
            v *= scale[a];
        }
        low[i] = v;
    }
}

}  // namespace

int pack_rows(const uint16_t* src, int64_t ld, int64_t rows, int64_t k, uint16_t* dst, int64_t kp, hipStream_t st) {
    const int64_t groups = (rows * (kp / 8) + 255) / 256;
    hipLaunchKernelGGL(k_pack, dim3((unsigned)(groups < 8192 ? groups : 8192)), dim3(256), 0, st, src, ld, rows, k, dst, kp);
    SPA_HIP_TRY(hipGetLastError());
    return SPA_OK;
}

int half_rows(const uint16_t* src, int kind, int64_t ld, int64_t rows, int64_t k, uint16_t* dst, int64_t kp, int64_t ldd, int32_t* e,
              float* norm, bool twice, hipStream_t st) {
    const dim3 grid((unsigned)rows);
    if (kp <= 4096) hipLaunchKernelGGL((k_half_rows<16, 256>), grid, dim3(256), 0, st, src, kind, ld, k, dst, kp, ldd, e, norm, twice);
    else if (kp <= 16384) hipLaunchKernelGGL((k_half_rows<16, 1024>), grid, dim3(1024), 0, st, src, kind, ld, k, dst, kp, ldd, e, norm, twice);
    else hipLaunchKernelGGL((k_half_rows<0, 1024>), grid, dim3(1024), 0, st, src, kind, ld, k, dst, kp, ldd, e, norm, twice);
    SPA_HIP_TRY(hipGetLastError());
    return SPA_OK;
}

int half_blocks(int type, const uint8_t* src, int64_t rows, int64_t k, uint16_t* dst, int64_t kp, int64_t ldd, int32_t* e, float* norm,
                bool rest, hipStream_t st) {
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
#define SPA_BLOCKS_TILE(T, QK, BS, TILE, FULL)                                                                          \
    hipLaunchKernelGGL((k_half_blocks<T, QK, BS, TILE, FULL>), dim3((unsigned)rows), dim3(256), 0, st, src, k, dst, kp, ldd, e, norm, rest, t, align)
#define SPA_BLOCKS_FORM(T, QK, BS)                                                                                      \
    do {                                                                                                                \
        if (k <= 4096 && (norm || rest)) SPA_BLOCKS_TILE(T, QK, BS, 4096, true);                                        \
        else if (k <= 4096) SPA_BLOCKS_TILE(T, QK, BS, 4096, false);                                                    \
        else if (norm || rest) SPA_BLOCKS_TILE(T, QK, BS, 16384, true);                                                 \
        else SPA_BLOCKS_TILE(T, QK, BS, 16384, false);                                                                  \
    } while (0)
    switch (type) {
#define SPA_BLOCKS(T, QK, BS)                                                                                           \
    case T:                                                                                                             \
        SPA_BLOCKS_FORM(T, QK, BS);                                                                                     \
        break;
        SPA_BLOCKS(2, 32, 18) SPA_BLOCKS(3, 32, 20) SPA_BLOCKS(6, 32, 22) SPA_BLOCKS(7, 32, 24) SPA_BLOCKS(8, 32, 34)
        SPA_BLOCKS(10, 256, 84) SPA_BLOCKS(11, 256, 110) SPA_BLOCKS(12, 256, 144) SPA_BLOCKS(13, 256, 176) SPA_BLOCKS(14, 256, 210)
        SPA_BLOCKS(16, 256, 66) SPA_BLOCKS(17, 256, 74) SPA_BLOCKS(18, 256, 98) SPA_BLOCKS(19, 256, 50) SPA_BLOCKS(20, 32, 18)
        SPA_BLOCKS(21, 256, 110) SPA_BLOCKS(22, 256, 82) SPA_BLOCKS(23, 256, 136) SPA_BLOCKS(29, 256, 56) SPA_BLOCKS(42, 64, 18)
#undef SPA_BLOCKS
#undef SPA_BLOCKS_FORM
#undef SPA_BLOCKS_TILE
        default: return fail(SPA_ERR_TYPE, "weights of type %d are not supported", type);
    }
    SPA_HIP_TRY(hipGetLastError());
    return SPA_OK;
}

int transpose16(const uint16_t* src, int64_t ld, int64_t rows, int64_t cols, uint16_t* dst, int64_t ldd, int64_t rp,
                const int32_t* re, const int32_t* ce, hipStream_t st) {
    const int64_t tr = (rp + 63) / 64, tc = (cols + 63) / 64;
    const dim3 grid((unsigned)(tr * tc));
    if (re) hipLaunchKernelGGL((k_transpose<true>), grid, dim3(256), 0, st, src, ld, rows, cols, dst, ldd, rp, tc, re, ce);
    else hipLaunchKernelGGL((k_transpose<false>), grid, dim3(256), 0, st, src, ld, rows, cols, dst, ldd, rp, tc, re, ce);
    SPA_HIP_TRY(hipGetLastError());
    return SPA_OK;
}

int norms16(const uint16_t* x, int64_t ldx, int64_t m, const uint16_t* w0, const uint16_t* w1, int64_t n, int64_t k, float* xn, float* n0,
            float* n1, hipStream_t st) {
    hipLaunchKernelGGL(k_norms, dim3((unsigned)(m + 2 * n)), dim3(256), 0, st, Norms{x, w0, w1, ldx, m, n, k, xn, n0, n1});
    SPA_HIP_TRY(hipGetLastError());
    return SPA_OK;
}

int64_t top_run(int64_t m) {
    const int64_t r = (m + TOP_PIECES - 1) / TOP_PIECES;
    return r < TOP_RUN ? TOP_RUN : r;
}
int64_t tops_part(int64_t m, int64_t n) {
    const int64_t np = (n + 63) / 64 * 64;
    return (n + TOP_COLS - 1) / TOP_COLS * m + (m + top_run(m) - 1) / top_run(m) * np;
}
int tops16(const uint16_t* dh, int64_t ld, int64_t m, int64_t n, const float* xn, const float* n0, const float* n1, float* part, int32_t* ge,
           int32_t* ce, hipStream_t st) {
    Tops q{};
    q.dh = dh;
    q.ld = ld;
    q.m = m;
    q.n = n;
    q.np = (n + 63) / 64 * 64;
    q.run = top_run(m);
    q.xn = xn;
    q.n0 = n0;
    q.n1 = n1;
    q.tiles = (int)((n + TOP_COLS - 1) / TOP_COLS);
    q.pieces = (int)((m + q.run - 1) / q.run);
    q.rows = part;
    q.cols = part + q.tiles * m;
    q.ge = ge;
    q.ce = ce;
    const dim3 grid((unsigned)q.tiles, (unsigned)q.pieces);
    if (ld % 2 == 0 && (reinterpret_cast<uintptr_t>(dh) & 3) == 0) hipLaunchKernelGGL((k_tops<true>), grid, dim3(256), 0, st, q);
    else hipLaunchKernelGGL((k_tops<false>), grid, dim3(256), 0, st, q);
    SPA_HIP_TRY(hipGetLastError());
    hipLaunchKernelGGL(k_exponents, dim3((unsigned)((m + q.np + 255) / 256)), dim3(256), 0, st, q);
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
             const int32_t* which, int pool, int rank, float* low, int rp, const Frags& fr, hipStream_t st) {
    const bool words = k % 2 == 0 && ldx % 2 == 0 && ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(a)) & 3) == 0;
    // two tiles of four, whose loads begin anywhere, do not fit in the registers
    const int64_t rows = m > 256 && (words || rp <= 16) ? 32 : 16, tiles = (m + rows - 1) / rows;
    const int most = pool < rows ? pool : (int)rows;
    int64_t more = 0;                                             // two fragments a lane
    if (fr.out) more = ((int64_t)fr.tiles * (fr.k / 32) * 64 + tiles * LOW_WAVES * 128 - 1) / (tiles * LOW_WAVES * 128);
    if (more > 256) more = 256;
    const dim3 grid((unsigned)tiles, (unsigned)(most + more)), block(LOW_WAVES * 64);
#define SPA_LOW(KIND, MT, TILES, WORDS)                                                                                       \
    hipLaunchKernelGGL((k_low<KIND, MT, TILES, WORDS>), grid, block, 0, st, x, ldx, m, k, a, scale, which, pool, rank, low, \
                       rp, most, fr)
#define SPA_LOW_ROWS(KIND)                                           \
    do {                                                             \
        if (rows == 32 && rp > 16) SPA_LOW(KIND, 2, 4, true);        \
        else if (rows == 32 && words) SPA_LOW(KIND, 2, 1, true);     \
        else if (rows == 32) SPA_LOW(KIND, 2, 1, false);             \
        else if (rp <= 16 && words) SPA_LOW(KIND, 1, 1, true);       \
        else if (rp <= 16) SPA_LOW(KIND, 1, 1, false);               \
        else if (words) SPA_LOW(KIND, 1, 4, true);                   \
        else SPA_LOW(KIND, 1, 4, false);                             \
    } while (0)
    if (kind == SRC_BF16) SPA_LOW_ROWS(SRC_BF16);
    else SPA_LOW_ROWS(SRC_F16);
#undef SPA_LOW_ROWS
#undef SPA_LOW
    SPA_HIP_TRY(hipGetLastError());
    return SPA_OK;
}

int low_pick(const float* part, int pieces, const float* scale, const int32_t* which, int64_t m, int pool, int rank, float* low, int rp,
             hipStream_t st) {
    const int64_t groups = (m * rp + 255) / 256;
    hipLaunchKernelGGL(k_low_pick, dim3((unsigned)(groups < 4096 ? groups : 4096)), dim3(256), 0, st, part, pieces, scale, which, m, pool, rank, low, rp);
    SPA_HIP_TRY(hipGetLastError());
    return SPA_OK;
}

}  // namespace lin
}  // namespace spa
