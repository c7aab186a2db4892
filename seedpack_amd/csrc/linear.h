// Products with packed weights: what their kernels share (gemm.hip, few.hip, rows.hip, linear.hip).
//
// Numbers. Every sum is held in 32 bits. Where the inputs and the weights have the same 16-bit type
// their products are exact in float32 and go through that type's matrix instruction. Where they do not
// (block types, BF16 beside F16) there are two forms:
//   * many rows: both operands as binary16 with a power of two taken out of each row, so that the row's
//     largest value lies below 2^15. A row of 16-bit numbers keeps its values to 2^-39 of its largest (2^-24 is the
//     least step), one of blocks to 2^-34; a decoded weight is rounded to 11 bits, an eighth of a BF16
//     rounding: an output's own rounding is eight times that, and 22 bits would take the product twice as long. Beside
//     F16 inputs, whose results have 11 bits too, the weights are taken to 22: what the rounding leaves over
//     takes part as a second half of k. The powers are added back to the float32 sums as exponents;
//   * few rows: whole codes of five block types as they are (codes.hip), each value of the others as a sum of two
//     BF16 numbers (16 bits, any exponent), whose products are summed by two or three BF16 instructions: the
//     matrix unit idles there.
#pragma once

#include "common.h"

namespace spa {
namespace lin {

typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 hf8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));

// the 16-bit types of the products' inputs (SRC_BF16 / SRC_F16)
__device__ __forceinline__ float wide(uint32_t h, int kind) {
    if (kind == SRC_BF16) return bf16_to_f32(h);
    return (float)__builtin_bit_cast(_Float16, (uint16_t)h);
}
__device__ __forceinline__ uint16_t narrow(float v, int kind) {
    if (kind == SRC_BF16) return __builtin_bit_cast(uint16_t, (__bf16)v);
    return __builtin_bit_cast(uint16_t, (_Float16)v);
}
__device__ __forceinline__ uint32_t narrow2(float a, float b, int kind) {
    return (uint32_t)narrow(a, kind) | ((uint32_t)narrow(b, kind) << 16);
}
// Eight 16-bit numbers from any number's address, by whole aligned words (each holds at least one of them): 16-byte
// loads that begin between words take several times as long as others.
__device__ __forceinline__ u4 load8_words(const uint16_t* p) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    const uint32_t* w = reinterpret_cast<const uint32_t*>(at & ~(uintptr_t)3);
    const uint32_t odd = (uint32_t)at & 2;
    u4 v;
    __builtin_memcpy(&v, w, 16);
    const uint32_t t = w[odd ? 4 : 3];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __builtin_amdgcn_alignbyte(i < 3 ? v[i + 1] : t, v[i], odd);
    return v;
}

// two binary16 numbers beside the second parts of weights: infinities as zeros. Beside the first parts they have
// made the sum infinite, and a second part may be zero.
__device__ __forceinline__ uint32_t finite2(uint32_t h) {
    return h & (((h & 0x7fffu) == 0x7c00u ? 0u : 0xffffu) | ((h & 0x7fff0000u) == 0x7c000000u ? 0u : 0xffff0000u));
}

// v = hi + lo to 2^-17 of v: hi is v cut to BF16 (so that v - hi is exact), lo the rest rounded.
// Infinities and NaN stay in hi alone.
__device__ __forceinline__ void split8(const float (&v)[8], bf8& hi, bf8& lo) {
    u4 h;
    bf8 l;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t a = __float_as_uint(v[2 * i]), b = __float_as_uint(v[2 * i + 1]);
        // a NaN whose payload lies in the cut bits would become an infinity: its quiet bit is set
        const uint32_t ah = v[2 * i] == v[2 * i] ? a : (a | 0x400000u), bh = v[2 * i + 1] == v[2 * i + 1] ? b : (b | 0x400000u);
        h[i] = __builtin_amdgcn_perm(bh, ah, 0x07060302u);
        const bool fa = (a & 0x7f800000u) != 0x7f800000u, fb = (b & 0x7f800000u) != 0x7f800000u;
        l[2 * i] = (__bf16)(fa ? v[2 * i] - __uint_as_float(a & 0xffff0000u) : 0.f);
        l[2 * i + 1] = (__bf16)(fb ? v[2 * i + 1] - __uint_as_float(b & 0xffff0000u) : 0.f);
    }
    hi = __builtin_bit_cast(bf8, h);
    lo = l;
}

// A gate's value and slope. silu: g s(g), s the logistic; gelu in its tanh form,
// 0.5 g (1 + tanh(t)) = g s(2t), t = sqrt(2/pi) (g + 0.044715 g^3).
enum Act { ACT_SILU = 0, ACT_GELU = 1 };
__device__ __forceinline__ float act_logit(float g, int act) {
    return act == ACT_SILU ? g : 1.5957691216057308f * (g + 0.044715f * g * g * g);
}
// e^-t: the exponent in units of log2 as a sum of two floats, so that the product's rounding does not grow with t;
// the hardware's 2^x and 1/x are good to an ulp. (expf and a division of full IEEE rounding: 131 us instead of 115
// for a round of 256 x 256 tiles of the gated product, k = 4096.) Where it overflows its reciprocal is zero.
__device__ __forceinline__ float exp_minus(float t) {
    const float h = -1.44269504f * t, l = fmaf(-1.44269504f, t, -h) - 1.92596303e-8f * t;
    const float e = __builtin_amdgcn_exp2f(h), r = fmaf(e * 0.69314718f, l, e);
    return r == r ? r : e;                                        // infinite t or e
}
__device__ __forceinline__ float act_value(float g, int act) {
    return g * __builtin_amdgcn_rcpf(1.f + exp_minus(act_logit(g, act)));
}
__device__ __forceinline__ void act_both(float g, int act, float& value, float& slope) {
    const float e = exp_minus(act_logit(g, act)), p = __builtin_amdgcn_rcpf(1.f + e);
    const float dt = act == ACT_SILU ? 1.f : 1.5957691216057308f * (1.f + 0.134145f * g * g);
    const float q = p * fminf(e * p, 1.f);                        // p (1 - p) without the difference; e may be infinite
    value = g * p;
    // q is zero long before g^2 overflows: zero times a large g is zero
    slope = p + (q > 0.f ? g * q * dt : 0.f * g);
}

// the adapters of a call: low[m][rp] = s_a x[m] A_a^T in float32 (rp = the rank rounded up to 16, zeros
// beyond it), b the adapters' second matrices
struct Expand {
    const float* low;
    const uint16_t* b;        // [pool][n][rank], the type of the inputs
    const int32_t* which;     // [m]; a row whose number is outside 0..pool-1 has none
    int pool, rank, rp, kind;
    bool wide_b;              // 16-byte loads of b's rows: rank a multiple of 8, b 16-byte aligned
};

// the adapters' part of output (m, n) of `count` columns
__device__ __forceinline__ float expand(const Expand& ex, int m, int n, int count) {
    const int a = ex.which[m];
    if (a < 0 || a >= ex.pool) return 0.f;
    const float* z = ex.low + (int64_t)m * ex.rp;
    const uint16_t* b = ex.b + ((int64_t)a * count + n) * ex.rank;
    float t = 0.f;
    if (ex.wide_b) {
        for (int r = 0; r < ex.rank; r += 8) {
            const u4 h = *reinterpret_cast<const u4*>(b + r);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                t = fmaf(z[r + 2 * c], wide(h[c] & 0xffffu, ex.kind), t);
                t = fmaf(z[r + 2 * c + 1], wide(h[c] >> 16, ex.kind), t);
            }
        }
    } else {
        for (int r = 0; r < ex.rank; r += 8) {                    // eight loads at once; those beyond the last are dropped
            uint16_t h[8];
#pragma unroll
            for (int c = 0; c < 8; ++c) h[c] = b[tmin(r + c, ex.rank - 1)];
#pragma unroll
            for (int c = 0; c < 8; ++c) t = r + c < ex.rank ? fmaf(z[r + c], wide(h[c], ex.kind), t) : t;
        }
    }
    return t;
}

// OUT_PART: a piece of k in float32 (joined by a launch of its own into any of the others); OUT_LOW: plain, and the adapters' second product
enum GemmOut { OUT_PLAIN = 0, OUT_GATED = 1, OUT_GRAD = 2, OUT_LOW = 3, OUT_PART = 4 };
constexpr int GEMM_PIECES = 16;

// The inputs as the few-rows products' matrix instruction takes them: for each step of 32 k and each tile of 16 rows
// a run of 64 lanes x 8 numbers, one contiguous load of a wave. halves: tiles of 8 rows, each there twice, with the
// first 16 k of a step and with the second. k a multiple of 32, rows at 16-byte addresses.
struct Frags {
    uint16_t* out;            // null: none
    int tiles, k;
    bool halves;
};
__device__ __forceinline__ void fragment(const Frags& fr, const uint16_t* x, int64_t ldx, int64_t m, int i) {
    const int lane = i & 63, tile = (i >> 6) % fr.tiles, step = (i >> 6) / fr.tiles;
    const int row = lane & 15, g = lane >> 4, r = fr.halves ? 8 * tile + (row & 7) : 16 * tile + row;
    u4 v = {0, 0, 0, 0};
    if (r < m && (!fr.halves || (row < 8) == (g < 2))) v = *reinterpret_cast<const u4*>(x + (int64_t)r * ldx + step * 32 + 8 * g);
    reinterpret_cast<u4*>(fr.out)[i] = v;
}

// sum_k x[m][k] w[n][k] over rows padded to a multiple of 64 (zeros), and what becomes of it
struct Gemm {
    int half;                 // SRC_BF16 / SRC_F16: the type of both operands
    const uint16_t* x;        // [m][k], rows of ldx, 16-byte aligned
    const uint16_t *w0, *w1;  // [n][k], rows of ldw; w1: the second matrix of OUT_GATED / OUT_GRAD
    int64_t ldx, ldw;
    int m, n, k;
    const int32_t *xe, *we0, *we1;   // powers of two taken out of the rows, or null
    int kind;                 // type of y and dh
    uint16_t* y;              // [m][n], rows of ldy (not OUT_GRAD)
    int64_t ldy;
    Expand ex;                // OUT_LOW (ex.low null: OUT_PLAIN)
    int act;
    const uint16_t* dh;       // OUT_GRAD: [m][n], rows of ldh
    int64_t ldh;
    uint16_t* grad;           // OUT_GRAD: [m][2 np], the gate's gradient, then the up projection's; zeros beyond n
    int64_t np, ldg;          // its halves' width and its rows' distance
    bool twice;               // OUT_GRAD: grad's columns again, 2 np further on
    const int32_t* ge;        // OUT_GRAD: power of two taken out of each row of grad (binary16), or null
    // pieces of k: the most that there may be (1: none), scratch of gemm_part() numbers for their sums
    // [matrix][piece][m][n], and how many there are
    int most;
    float* part;
    int pieces;
    const int32_t* which;     // gemm_pieces: weight row n serves the rows m with which[m] = n / rank only, or null
    int rank;
};
int64_t gemm_part(const Gemm& g);
// what a product is expected to take, in hundredths of a microsecond
int64_t gemm_cost(const Gemm& g);
// the pieces alone, left in part as [piece][m][n]; g.pieces of them
int gemm_pieces(const Gemm& g, hipStream_t st);
int gemm(const Gemm& g, hipStream_t st);

// ---- few rows (few.hip)
struct Few {
    int type;                 // the weights' ggml type (1 F16, 30 BF16, or a block type)
    const uint8_t *w0, *w1;   // w1 for the gated form, else null
    int64_t wbytes;           // bytes of each matrix
    int64_t rowbytes;         // and of a row of it
    int n, k;                 // k: whole steps of 32, x zero beyond the weights' own
    const uint16_t* x;        // [m][k], rows of ldx (a multiple of 8), 16-byte aligned
    int64_t ldx;
    int m, kind;
    uint16_t* y;
    int64_t ldy;
    Expand ex;
    int act;
    bool framed;              // frags holds the inputs' fragments already
};
constexpr int FEW_ROWS = 64;
// frags: scratch of few_fragments numbers
int few(const Few& f, uint16_t* frags, hipStream_t st);
// types whose codes go to the matrix unit as they are (codes.hip)
inline bool coded(int type) { return type == 2 || type == 8 || type == 12 || type == 13 || type == 14; }
int few_codes(const Few& f, uint16_t* frags, hipStream_t st);
// tiles of input rows: 16 rows each, or 8 (Q6_K), a power of two of them
inline int few_tiles(int type, int64_t m) {
    int t = 1;
    while (t * (type == 14 ? 8 : 16) < m) t *= 2;
    return t;
}
inline int64_t few_fragments(int type, int64_t m, int64_t kp) {
    return (coded(type) || type == 1 || type == 30) && few_tiles(type, m) > 1 ? few_tiles(type, m) * 16 * kp : 0;
}
// the most rows that take the few-rows form, FEW_ROWS at a time: where codes are cheap to unpack twice is less than
// decoding the weights for the many-rows form (Q8_0 12288 x 4096: 28 us for 64 rows, 68 for 65 in the other form)
inline int64_t few_limit(int type) { return coded(type) && type != 14 ? 2 * FEW_ROWS : FEW_ROWS; }

// ---- rows (rows.hip)
// rows of a 16-bit matrix copied into rows of kp (a multiple of 64), zeros beyond k
int pack_rows(const uint16_t* src, int64_t ld, int64_t rows, int64_t k, uint16_t* dst, int64_t kp, hipStream_t st);
// the same into binary16, rows of ldd, with a power of two taken out of each row (e), and the row's 2-norm as it was (or
// null); twice: the row again kp further on
int half_rows(const uint16_t* src, int kind, int64_t ld, int64_t rows, int64_t k, uint16_t* dst, int64_t kp, int64_t ldd, int32_t* e,
              float* norm, bool twice, hipStream_t st);
// the same from a block type; rest: what the rounding leaves over kp further on
int half_blocks(int type, const uint8_t* src, int64_t rows, int64_t k, uint16_t* dst, int64_t kp, int64_t ldd, int32_t* e, float* norm,
                bool rest, hipStream_t st);
// dst[c][r] = src[r][c], rows of ldd, r padded with zeros to rp (rp and ldd multiples of 8); with re and ce F16 values
// times 2^(re[r] - ce[c])
int transpose16(const uint16_t* src, int64_t ld, int64_t rows, int64_t cols, uint16_t* dst, int64_t ldd, int64_t rp,
                const int32_t* re, const int32_t* ce, hipStream_t st);
// the power of two to take out of each row of the gated block's inner gradients, by the 2-norms of the inputs'
// rows and of both matrices' rows; top: 8 bytes of scratch
int grad_exponents(const uint16_t* dh, int kind, int64_t ld, int64_t rows, int64_t n, const float* xnorm, const float* n0,
                   const int32_t* e0, const float* n1, const int32_t* e1, void* top, int32_t* e, hipStream_t st);
// the 2-norms of the rows of x and of both matrices (F16)
int norms16(const uint16_t* x, int64_t ldx, int64_t m, const uint16_t* w0, const uint16_t* w1, int64_t n, int64_t k, float* xn, float* n0,
            float* n1, hipStream_t st);
// and the powers of two to take out of each row of the inner gradients, ge, and of each column, ce [gate np][up np], np
// the next multiple of 64; part: scratch of tops_part(m, n) numbers
int64_t tops_part(int64_t m, int64_t n);
int tops16(const uint16_t* dh, int64_t ld, int64_t m, int64_t n, const float* xn, const float* n0, const float* n1, float* part, int32_t* ge,
           int32_t* ce, hipStream_t st);
int zero_rows(uint16_t* p, int64_t ld, int64_t rows, int64_t k, hipStream_t st);
// low[m][rp] = scale[a] x[m] A_a^T, a = which[m]; with fr.out the same launch writes the rows' fragments
int low_rows(const uint16_t* x, int64_t ldx, int kind, int64_t m, int64_t k, const uint16_t* a, const float* scale,
             const int32_t* which, int pool, int rank, float* low, int rp, const Frags& fr, hipStream_t st);

// the same from the pieces of x [A_0; A_1; ..]^T (gemm_pieces)
int low_pick(const float* part, int pieces, const float* scale, const int32_t* which, int64_t m, int pool, int rank, float* low, int rp,
             hipStream_t st);

}  // namespace lin
}  // namespace spa
