// Numbers to 4-bit floating point in microscaled blocks, and back.
//
// A block's scale is 2^e, e = floor(log2(its largest magnitude)) - 2 and not below -127, so that the largest lies
// in [4, 8) units; each number is rounded to the nearest of the grid, ties to the even code, and held at 6 units (the
// microscaling formats' published rule). The hardware's conversions do exactly that for every float and every scale.
// e comes from the float's exponent field: the scale's byte is that field less 2.
//
// Bound by memory: four lanes share a block, eight numbers each (16 bytes of 16-bit numbers a lane), and change
// their codes between pairs of lanes, so that loads and stores both are whole lines.
#include "../../include/seedpack_amd.h"
#include "lanes.h"
#include "launch.h"
#include "mx4.h"

#include <math.h>

namespace spa {
namespace mx {
namespace {

typedef uint32_t u4v __attribute__((ext_vector_type(4)));
typedef float f2 __attribute__((ext_vector_type(2)));

template <int KIND> __device__ __forceinline__ float wide_at(const void* p, int64_t i) {
    if constexpr (KIND == SRC_F32) return static_cast<const float*>(p)[i];
    else return lin::wide(static_cast<const uint16_t*>(p)[i], KIND);
}
template <int KIND> __device__ __forceinline__ void put(void* p, int64_t i, float v) {
    if constexpr (KIND == SRC_F32) static_cast<float*>(p)[i] = v;
    else static_cast<uint16_t*>(p)[i] = lin::narrow(v, KIND);
}

// the scale's byte of a block whose largest magnitude is `top`
__device__ __forceinline__ uint32_t scale_byte(float top) {
    const int field = (int)(__float_as_uint(top) >> 23);
    return field == 255 ? 255u : (uint32_t)tmax(field - 2, 0);
}
// the largest magnitude; infinities and NaN stay above all
__device__ __forceinline__ float larger(float a, float b) {
    return __uint_as_float(tmax(__float_as_uint(a) & 0x7fffffffu, __float_as_uint(b) & 0x7fffffffu));
}
// eight numbers' codes, the first lowest; a block of NaN has codes 0
__device__ __forceinline__ uint32_t codes8(const float (&x)[8], uint32_t byte) {
    const float scale = __uint_as_float(byte << 23);
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[0], x[1], scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[2], x[3], scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[4], x[5], scale, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[6], x[7], scale, 3);
    return byte == 255 ? 0u : c;
}
// four codes in the low halves of four bytes
__device__ __forceinline__ uint32_t spread(uint32_t v) {
    v = (v | v << 8) & 0x00ff00ffu;
    return (v | v << 4) & 0x0f0f0f0fu;
}

// eight numbers of a row at column c, zeros behind its last
template <int KIND> __device__ __forceinline__ void load8(const void* x, int64_t at, int64_t left, bool wide, float (&v)[8]) {
    if (left >= 8) {
        if constexpr (KIND == SRC_F32) {
            __builtin_memcpy(v, static_cast<const float*>(x) + at, 32);   // at any number's address
        } else {
            const uint16_t* const p = static_cast<const uint16_t*>(x) + at;
            const u4v a = wide ? *reinterpret_cast<const u4v*>(p) : lin::load8_words(p);
#pragma unroll
            for (int c = 0; c < 8; ++c) v[c] = lin::wide((a[c >> 1] >> (16 * (c & 1))) & 0xffffu, KIND);
        }
    } else {
#pragma unroll
        for (int c = 0; c < 8; ++c) v[c] = c < left ? wide_at<KIND>(x, at + c) : 0.f;
    }
}

struct Rows {
    const void* x;
    int64_t rows, cols, stride;
    int pitch;
    bool wide;
    uint8_t *codes, *scales;
};

template <int KIND>
__global__ __launch_bounds__(256) void k_quantize(const Rows a) {
    const int64_t per = (int64_t)a.pitch * 4, id = blockIdx.x * 256ll + threadIdx.x;
    const int64_t row = id / per;
    if (row >= a.rows) return;                                    // whole blocks of lanes: per is a multiple of 4
    const int64_t quarter = id - row * per, c = quarter * 8;
    float v[8];
    load8<KIND>(a.x, row * a.stride + c, a.cols - c, a.wide, v);
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = larger(top, v[i]);
    top = larger(top, lane_move<0xb1>(top));
    top = larger(top, lane_move<0x4e>(top));
    const uint32_t byte = scale_byte(top), mine = codes8(v, byte), other = moved<0x4e>(mine);
    // lanes 0 and 2 hold numbers 0-7 and 16-23 of the block: bytes 0-7; lanes 1 and 3 the rest
    const int q = threadIdx.x & 3;
    const bool upper = q >= 2;
    const uint32_t lo = upper ? other >> 16 : mine & 0xffffu, hi = upper ? mine >> 16 : other & 0xffffu;
    const int64_t block = id >> 2;
    reinterpret_cast<uint32_t*>(a.codes)[block * 4 + (q & 1) * 2 + (q >> 1)] = spread(lo) | spread(hi) << 4;
    if (q == 0) a.scales[block] = (uint8_t)byte;
}

// Blocks along columns: the matrix of x^T. A workgroup takes 64 columns of 256 rows, a lane a column of 32 of them; the
// codes leave by way of LDS, 128 bytes of a column at a time. Neighbouring columns are of one XCD, which takes every
// eighth workgroup: where rows begin at any address, their runs of 64 numbers share lines (2053 x 7169 float32: 88 MB read
// and 17.4 us with the columns dealt in turn, 59 and 14.0 so).
template <int KIND>
__global__ __launch_bounds__(512) void k_quantize_across(const Rows a) {
    __shared__ __align__(16) uint32_t codes[64][33];
    __shared__ uint8_t scales[64][8];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t strips = (uint32_t)((a.cols + 63) / 64), xcd = blockIdx.x & 7;
    const uint32_t tile = xcd * (gridDim.x / 8) + tmin(xcd, gridDim.x % 8) + (blockIdx.x >> 3), piece = tile / strips;
    const int64_t c0 = (int64_t)(tile - piece * strips) * 64, c = c0 + lane, r0 = (int64_t)piece * 256 + wave * 32;
    const bool in = c < a.cols;
    float v[32], top = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = in && r0 + i < a.rows ? wide_at<KIND>(a.x, (r0 + i) * a.stride + c) : 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) top = larger(top, v[i]);
    const uint32_t byte = scale_byte(top);
    uint32_t q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float part[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) part[j] = v[8 * i + j];
        q[i] = codes8(part, byte);
    }
    codes[lane][wave * 4 + 0] = spread(q[0] & 0xffffu) | spread(q[2] & 0xffffu) << 4;
    codes[lane][wave * 4 + 1] = spread(q[0] >> 16) | spread(q[2] >> 16) << 4;
    codes[lane][wave * 4 + 2] = spread(q[1] & 0xffffu) | spread(q[3] & 0xffffu) << 4;
    codes[lane][wave * 4 + 3] = spread(q[1] >> 16) | spread(q[3] >> 16) << 4;
    scales[lane][wave] = (uint8_t)byte;
    __syncthreads();
    for (int u = threadIdx.x; u < 64 * 32; u += 512) {
        const int64_t to = c0 + u / 32;
        if (to < a.cols) reinterpret_cast<uint32_t*>(a.codes)[(to * a.pitch + piece * 8) * 4 + u % 32] = codes[u / 32][u % 32];
    }
    for (int u = threadIdx.x; u < 64 * 8; u += 512) {
        const int64_t to = c0 + u / 8;
        if (to < a.cols) a.scales[to * a.pitch + piece * 8 + u % 8] = scales[u / 8][u % 8];
    }
}

struct Values {
    const uint8_t *codes, *scales;
    int64_t rows, cols, stride;
    int pitch;
    void* y;
};

// A lane takes eight neighbours of a block: the low or the high halves of eight bytes, brought together two to a byte
template <int KIND>
__global__ __launch_bounds__(256) void k_values(const Values a) {
    const int64_t per = (a.cols + 31) / 32 * 4, id = blockIdx.x * 256ll + threadIdx.x;
    const int64_t row = id / per;
    if (row >= a.rows) return;
    const int64_t eighth = id - row * per, block = row * a.pitch + (eighth >> 2), c = eighth * 8, left = a.cols - c;
    if (left <= 0) return;
    const int q = (int)(eighth & 3);
    const lin::u2 v = reinterpret_cast<const lin::u2*>(a.codes)[block * 2 + (q & 1)];
    const float scale = __uint_as_float((uint32_t)a.scales[block] << 23);
    float x[8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t m = (v[h] >> (4 * (q >> 1))) & 0x0f0f0f0fu, both = m | m >> 4;
        const f2 lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(both, scale, 0), hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(both, scale, 2);
        x[4 * h] = lo[0];
        x[4 * h + 1] = lo[1];
        x[4 * h + 2] = hi[0];
        x[4 * h + 3] = hi[1];
    }
    const int64_t at = row * a.stride + c;
    if (left >= 8) {
        // at any number's address
        if constexpr (KIND == SRC_F32) {
            __builtin_memcpy(static_cast<float*>(a.y) + at, x, 32);
        } else {
            const u4v w = {lin::narrow2(x[0], x[1], KIND), lin::narrow2(x[2], x[3], KIND), lin::narrow2(x[4], x[5], KIND), lin::narrow2(x[6], x[7], KIND)};
            __builtin_memcpy(static_cast<uint16_t*>(a.y) + at, &w, 16);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < left) put<KIND>(a.y, at + i, x[i]);
    }
}

// GGUF blocks, a scale's byte before 16 bytes of codes, taken apart: a lane 4 bytes of a block
__global__ __launch_bounds__(256) void k_from_blocks(const uint8_t* b, int64_t rows, int64_t blocks, int pitch, uint8_t* codes, uint8_t* scales) {
    const int64_t per = (int64_t)pitch * 4, id = blockIdx.x * 256ll + threadIdx.x, row = id / per;
    if (row >= rows) return;
    const int64_t block = (id - row * per) >> 2;
    const int q = threadIdx.x & 3;
    uint32_t v = 0;
    uint8_t s = 0;
    if (block < blocks) {
        const uint8_t* p = b + (row * blocks + block) * 17;
        __builtin_memcpy(&v, p + 1 + 4 * q, 4);
        s = p[0];
    }
    reinterpret_cast<uint32_t*>(codes)[id] = v;
    if (q == 0) scales[id >> 2] = s;
}

bool on(const void* p, uintptr_t unit) { return (reinterpret_cast<uintptr_t>(p) & (unit - 1)) == 0; }
constexpr int64_t MOST_COLS = 4000000;

int check_kind(const char* who, int kind) {
    if (kind != SPA_SRC_BF16 && kind != SPA_SRC_F16 && kind != SPA_SRC_F32) return fail(SPA_ERR_TYPE, "%s: numbers of kind %d (BF16, F16 and F32 are taken)", who, kind);
    return SPA_OK;
}
// a matrix of `rows` rows of `cols`; its codes and scales where given
int check_matrix(const char* who, int64_t rows, int64_t cols, const void* codes, const void* scales) {
    if (rows < 0 || cols < 1 || cols > MOST_COLS || rows > INT32_MAX - 1024 || rows * pitch_of(cols) * 4 / 256 >= INT32_MAX) return fail(SPA_ERR_ARG, "%s: bad shape %lld x %lld", who, (long long)rows, (long long)cols);
    if (rows && (!codes || !scales)) return fail(SPA_ERR_ARG, "%s: a pointer is NULL", who);
    if (!on(codes, 16) || !on(scales, 8)) return fail(SPA_ERR_ARG, "%s: codes have to be 16-byte aligned, scales 8-byte aligned", who);
    return SPA_OK;
}

// the workgroups of a conversion of rows x cols numbers, `threads` each
int check_launch(const char* who, int64_t workgroups, int threads, int64_t rows, int64_t cols) {
    if (!one_launch(workgroups, threads)) return fail(SPA_ERR_ARG, "%s: %lld x %lld numbers are more than one launch takes", who, (long long)rows, (long long)cols);
    return SPA_OK;
}

}  // namespace
}  // namespace mx
}  // namespace spa

using namespace spa;
using namespace spa::mx;

extern "C" {

int64_t spa_mx4_pitch(int64_t cols) { return cols < 1 || cols > MOST_COLS ? 0 : pitch_of(cols); }

int spa_mx4_quantize(const void* x, int kind, int64_t rows, int64_t cols, int64_t stride, int across, uint8_t* codes,
                     uint8_t* scales, void* stream) {
    if (int rc = check_kind("mx4_quantize", kind)) return rc;
    if (across && rows < 1) return fail(SPA_ERR_ARG, "mx4_quantize: columns of %lld numbers", (long long)rows);
    if (int rc = check_matrix("mx4_quantize", across ? cols : rows, across ? rows : cols, codes, scales)) return rc;
    if (cols < 1 || stride < cols) return fail(SPA_ERR_ARG, "mx4_quantize: rows of %lld at a stride of %lld", (long long)cols, (long long)stride);
    if (!rows) return SPA_OK;
    if (!x) return fail(SPA_ERR_ARG, "mx4_quantize: a pointer is NULL");
    Rows a{x, rows, cols, stride, (int)pitch_of(across ? rows : cols), on(x, 16) && stride % (kind == SPA_SRC_F32 ? 4 : 8) == 0, codes, scales};
    hipStream_t st = (hipStream_t)stream;
    if (across) {
        const int64_t workgroups = (cols + 63) / 64 * (a.pitch / 8);
        if (int rc = check_launch("mx4_quantize", workgroups, 512, rows, cols)) return rc;
        const dim3 grid((unsigned)workgroups);
        if (kind == SPA_SRC_BF16) hipLaunchKernelGGL(k_quantize_across<SRC_BF16>, grid, dim3(512), 0, st, a);
        else if (kind == SPA_SRC_F16) hipLaunchKernelGGL(k_quantize_across<SRC_F16>, grid, dim3(512), 0, st, a);
        else hipLaunchKernelGGL(k_quantize_across<SRC_F32>, grid, dim3(512), 0, st, a);
        SPA_HIP_TRY(hipGetLastError());
        return SPA_OK;
    }
    const int64_t workgroups = (rows * a.pitch * 4 + 255) / 256;
    if (int rc = check_launch("mx4_quantize", workgroups, 256, rows, cols)) return rc;
    const dim3 grid((unsigned)workgroups);
    if (kind == SPA_SRC_BF16) hipLaunchKernelGGL(k_quantize<SRC_BF16>, grid, dim3(256), 0, st, a);
    else if (kind == SPA_SRC_F16) hipLaunchKernelGGL(k_quantize<SRC_F16>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(k_quantize<SRC_F32>, grid, dim3(256), 0, st, a);
    SPA_HIP_TRY(hipGetLastError());
    return SPA_OK;
}

int spa_mx4_values(const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t cols, void* y, int kind, int64_t stride,
                   void* stream) {
    if (int rc = check_kind("mx4_values", kind)) return rc;
    if (int rc = check_matrix("mx4_values", rows, cols, codes, scales)) return rc;
    if (stride < cols) return fail(SPA_ERR_ARG, "mx4_values: rows of %lld at a stride of %lld", (long long)cols, (long long)stride);
    if (!rows) return SPA_OK;
    if (!y) return fail(SPA_ERR_ARG, "mx4_values: a pointer is NULL");
    Values a{codes, scales, rows, cols, stride, (int)pitch_of(cols), y};
    hipStream_t st = (hipStream_t)stream;
    const int64_t workgroups = (rows * ((cols + 31) / 32) * 4 + 255) / 256;
    if (int rc = check_launch("mx4_values", workgroups, 256, rows, cols)) return rc;
    const dim3 grid((unsigned)workgroups);
    if (kind == SPA_SRC_BF16) hipLaunchKernelGGL(k_values<SRC_BF16>, grid, dim3(256), 0, st, a);
    else if (kind == SPA_SRC_F16) hipLaunchKernelGGL(k_values<SRC_F16>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(k_values<SRC_F32>, grid, dim3(256), 0, st, a);
    SPA_HIP_TRY(hipGetLastError());
    return SPA_OK;
}

int spa_mx4_from_blocks(const void* blocks, int64_t rows, int64_t cols, uint8_t* codes, uint8_t* scales, void* stream) {
    if (int rc = check_matrix("mx4_from_blocks", rows, cols, codes, scales)) return rc;
    if (cols % 32) return fail(SPA_ERR_ARG, "mx4_from_blocks: rows of %lld are not whole blocks of 32", (long long)cols);
    if (!rows) return SPA_OK;
    if (!blocks) return fail(SPA_ERR_ARG, "mx4_from_blocks: a pointer is NULL");
    const int64_t pitch = pitch_of(cols), workgroups = (rows * pitch * 4 + 255) / 256;
    if (int rc = check_launch("mx4_from_blocks", workgroups, 256, rows, cols)) return rc;
    hipLaunchKernelGGL(k_from_blocks, dim3((unsigned)workgroups), dim3(256), 0, (hipStream_t)stream,
                       (const uint8_t*)blocks, rows, cols / 32, (int)pitch, codes, scales);
    SPA_HIP_TRY(hipGetLastError());
    return SPA_OK;
}

namespace {

// What a product takes, by the forms' times on one MI355X, in us:
//   FEW16, FEW32  16 x 16 and 32 x 32 outputs a wave: 2.9 for a launch; then rounds of 256 workgroups, each of which takes, for a MB
//                 of weights, 41 and 1.65 more for each input row of a tile (32 x 32: 62 and 0.5). Two matrices are 60 and 0.5 where the
//                 rounds follow one another; 32 x 32 won at none of 148 sizes of them and is not there
//   SMALL         128 x 128 tiles: 4.2 and 0.7 a step of 256 of k where a compute unit has one, 5 and 1.19 where it has two;
//                 in pieces of k, where there are too few tiles: 2 for the joining launch and 3.3 TB/s for its sums
//   LARGE         256 x 256 tiles, one to a compute unit: 8 and 1.75 a step, 1.25 with most units idle
// Tiles take no less than 3 and the weights' bytes at 5 TB/s, where few rows read 285 MB at 6 TB/s. Weights past the cache behind the
// L2s, us by rows, FEW16 FEW32 SMALL LARGE and SMALL in 2 and 4 pieces of k:
//   12288 x 4096    1: 7.1 9.7 12.6 17.9 11.8 11.7    16: 9.2 10.9 12.9 18.3 12.1 12.4    64: 28.6 17.7 14.1 20.2 14.7 14.8
//                 256: 110 62.5 16.5 30.6 24.4 34.7
//   12288 x 8192    1: 13.2 20.5 29.9 42.5 20.6 18.3  16: 18.6 25.0 30.2 43.1 20.9 18.7   32: 31.7 29.4 30.7 45.1 21.7 20.1
//   131072 x 4096   1: 47.6 71.6 56.4 61.6 63.6 72.9  16: 80.2 92.7 58.2 63.2 69.1 81.7
//   65536 x 8192    1: 55.3 89.3 68.0 69.9 58.6 63.2  16: 83.7 103 68.8 71.2 61.8 67.5
//   2048 x 16384   32: 11.4 20.9 39.6 58.9 24.5 16.0  64: 20.3 20.8 40.5 60.5 25.1 16.8 (in 8 pieces 13.6 and 15.2)
//   4096 x 4096    64: 11.6 7.7 13.2 19.7 11.5 11.5
//   2 x 12288 x 4096    1: 15.4 23.2 18.0 24.9 18.8 22.8    32: 31.3 26.6 18.6 26.1 20.4 25.2
// By expert the rows' spread is not known on the host: rows are taken to be dealt at random, and half of the experts that have any
// to end in a tile of their own. Tiles of few rows cost less than full ones, so rounds of them are not rounded up. Waves of few
// rows count tiles anew in each workgroup: 0.6 more for the launch and 0.3 a round, 0.9 of more than 64 experts.
//   32 of 4096 x 7168, by slots   4: 13.3 17.8 21.2 30.0 17.7 19.1   32: 57.9 79.6 77.6 93.0 71.6 72.4   512: 183 167 97.9 108 114 127
//   64 of 2 x 1536 x 2048         4: 7.3 9.5 9.3 12.3 10.4 11.6      32: 23.5 40.5 26.7 30.4 29.5 34.3   512: 65 96 48.6 52.3 63 78
// The choice is the best or within 15% of it at 385 of 400 sizes; the rest are calls of a few us and uneven spreads of rows.
enum Form { FEW16, FEW32, SMALL, LARGE };
struct Plan {
    int form, pieces;
};
Plan plan(int64_t m, int64_t n, int64_t pitch, int64_t experts, bool gated) {
    const double steps = (double)pitch / 8, sides = gated ? 2 : 1;
    const double used = experts ? experts * (1 - exp(-(double)m / experts)) : 1;
    const double read = 3 + 17e-6 * n * pitch * sides * used / 5;
    auto rows = [&](double t) { return experts ? fmax(used, m / t + used / 2) : ceil(m / t); };
    auto rounds = [&](double r) { return experts ? fmax(r, 1) : ceil(r); };
    auto few = [&](int tiles, double us, double us_row) {
        const double width = FEW_WAVES / few_split((int)pitch) * 16 * tiles, tall = rows(16 * tiles), in = fmin(16 * tiles, m / tall);
        const double turns = ceil(n / width) * tall / 256, whole = experts || turns >= 4 ? fmax(turns, 1) : ceil(turns), row = 17e-6 * pitch * sides;
        const double each = (us + us_row * in) * fmin(width, n) * row + (experts ? experts > 64 ? 0.9 : 0.3 : 0);
        return 2.9 + (experts ? 0.6 : 0) + fmax(each * whole, gated ? (60 + 0.5 * in) * width * row * turns : 0);
    };
    auto small = [&](double tiles, double k) { return fmax(tiles <= 256 ? 4.2 + tiles / 200 + 0.7 * k : rounds(tiles / 512) * (5 + 1.19 * k), read); };
    Plan best{FEW16, 1};
    double least = few(1, 41, 1.65);
    auto take = [&](int form, int pieces, double us) {
        if (us < least) {
            best = Plan{form, pieces};
            least = us;
        }
    };
    if (!gated) take(FEW32, 1, few(2, 62, 0.5));
    const double tiles = ceil(n * sides / 128.0) * rows(128);
    take(SMALL, 1, small(tiles, steps));
    for (int p = 2; p <= 8 && 2 * p <= steps; ++p)
        take(SMALL, p, small(tiles * p, ceil(steps / p)) + 2 + (double)m * n * 8 * p * sides / 3.3e6);
    const double large = ceil(n * sides / 256.0) * rows(256);
    take(LARGE, 1, fmax(rounds(large / 256) * (8 + (1.25 + 0.5 * fmin(large / 256, 1)) * steps), read));
    return best;
}
uint64_t part_bytes(const Plan& c, int64_t m, int64_t n, bool gated) {
    return c.pieces > 1 ? ((uint64_t)c.pieces * (gated ? 2 : 1) * m * n * 4 + 255) / 256 * 256 : 0;
}
int check_work(const char* who, const void* work, uint64_t have, uint64_t need) {
    if (need && (!work || !on(work, 256) || have < need))
        return fail(SPA_ERR_ARG, "%s: needs a 256-byte aligned workspace of %llu bytes, got %llu", who, (unsigned long long)need, (unsigned long long)(work ? have : 0));
    return SPA_OK;
}

// one of the products: checked, then launched
int product(const char* who, Product p, int64_t x_rows, int64_t k, int64_t n, int64_t experts, const int32_t* order, const int32_t* starts,
            int64_t slots, int64_t y_stride, void* work, uint64_t work_bytes, hipStream_t st) {
    if (int rc = check_kind(who, p.kind)) return rc;
    if (int rc = check_matrix(who, x_rows, k, p.xc, p.xs)) return rc;
    if (experts < 0 || experts > 1024 || n < 0 || n > INT32_MAX - 1024) return fail(SPA_ERR_ARG, "%s: %lld experts of %lld outputs (up to 1024 experts)", who, (long long)experts, (long long)n);
    if (int rc = check_matrix(who, n, k, p.w0c, p.w0s)) return rc;
    if ((p.w1c || p.w1s) && check_matrix(who, n, k, p.w1c, p.w1s)) return SPA_ERR_ARG;
    const int64_t m = experts ? slots : x_rows;
    if (m < 0 || m > INT32_MAX - 1024 || y_stride < n) return fail(SPA_ERR_ARG, "%s: bad shape %lld x %lld, stride %lld", who, (long long)m, (long long)n, (long long)y_stride);
    if (m == 0 || n == 0) return SPA_OK;
    if (!p.y) return fail(SPA_ERR_ARG, "%s: a pointer is NULL", who);
    p.pitch = (int)pitch_of(k);
    p.m = (int)m;
    p.n = (int)n;
    p.ldy = y_stride;
    p.each = 1;
    if (experts) {
        if (!order || !starts) return fail(SPA_ERR_ARG, "%s: order and starts are needed beside experts", who);
        if (x_rows == 0 || slots % x_rows) return fail(SPA_ERR_ARG, "%s: %lld slots of %lld rows", who, (long long)slots, (long long)x_rows);
        // rows are read at 32-bit offsets from the matrix's first
        if (x_rows * p.pitch * 16 >= (1ll << 32)) return fail(SPA_ERR_ARG, "%s: %lld rows of %lld by expert are more than 4 GiB of codes", who, (long long)x_rows, (long long)k);
        p.each = (int)(slots / x_rows);
        // 2^32 / each, rounded up by less than 1: exact where what slot times that adds stays below 1 / each
        p.magic = p.each > 1 && slots * p.each < (1ll << 32) ? (uint32_t)((1ull << 32) / p.each + 1) : 0;
        p.experts = (int)experts;
        p.order = order;
        p.starts = starts;
    }
    const Plan c = plan(p.m, p.n, p.pitch, p.experts, p.w1c != nullptr);
    if (int rc = check_work(who, work, work_bytes, part_bytes(c, p.m, p.n, p.w1c != nullptr))) return rc;
    p.pieces = c.pieces;
    p.part = (float*)work;
    return c.form <= FEW32 ? product_few(p, c.form == FEW32, st) : product_many(p, c.form == LARGE, st);
}

}  // namespace

uint64_t spa_mx4_product_work_bytes(int64_t x_rows, int64_t k, int64_t n, int64_t experts, int64_t slots, int gated) {
    const int64_t m = experts > 0 ? slots : x_rows;
    if (m <= 0 || m > INT32_MAX - 1024 || n <= 0 || n > INT32_MAX - 1024 || k < 1 || k > MOST_COLS || experts > 1024) return 0;
    return part_bytes(plan(m, n, pitch_of(k), experts > 0 ? experts : 0, gated), m, n, gated);
}

int spa_mx4_project(const uint8_t* x_codes, const uint8_t* x_scales, int64_t x_rows, int64_t k, const uint8_t* w_codes,
                    const uint8_t* w_scales, int64_t n, int64_t experts, const int32_t* order, const int32_t* starts, int64_t slots,
                    void* y, int y_kind, int64_t y_stride, void* work, uint64_t work_bytes, void* stream) {
    Product p{};
    p.xc = x_codes;
    p.xs = x_scales;
    p.w0c = w_codes;
    p.w0s = w_scales;
    p.y = y;
    p.kind = y_kind;
    return product("mx4_project", p, x_rows, k, n, experts, order, starts, slots, y_stride, work, work_bytes, (hipStream_t)stream);
}

int spa_mx4_gated(const uint8_t* x_codes, const uint8_t* x_scales, int64_t x_rows, int64_t k, const uint8_t* gate_codes,
                  const uint8_t* gate_scales, const uint8_t* up_codes, const uint8_t* up_scales, int64_t n, int act, int64_t experts,
                  const int32_t* order, const int32_t* starts, int64_t slots, void* h, int h_kind, int64_t h_stride, void* work,
                  uint64_t work_bytes, void* stream) {
    if (act != 0 && act != 1) return fail(SPA_ERR_ARG, "mx4_gated: unknown activation %d", act);
    if (n && (!up_codes || !up_scales)) return fail(SPA_ERR_ARG, "mx4_gated: a pointer is NULL");
    Product p{};
    p.xc = x_codes;
    p.xs = x_scales;
    p.w0c = gate_codes;
    p.w0s = gate_scales;
    p.w1c = up_codes;
    p.w1s = up_scales;
    p.act = act;
    p.y = h;
    p.kind = h_kind;
    return product("mx4_gated", p, x_rows, k, n, experts, order, starts, slots, h_stride, work, work_bytes, (hipStream_t)stream);
}

}  // extern "C"
