// Column sums of squares, per expert or whole: what an importance matrix gathers of a matrix's inputs
// (llama.cpp's "in_sum2" and "counts"). Bound by reading x once: 16384 x 12288 float32 136 us and 5 us of joining,
// 5.9 TB/s. By expert a row is read once for each of its experts: 16384 x 4096 BF16, two of 64, 53 and 8 us, 5.1 TB/s.
//
// A workgroup takes 512 columns (8 a lane, 64 lanes) and a run of rows, its four waves every fourth row of
// it; it joins the waves in LDS and writes one partial row, and a second launch adds the partial rows to the
// caller's sums in the order of the runs. Sums are float32; no atomics, so a call's result depends on its
// sizes only. With experts a workgroup belongs to one of them and takes that expert's rows of its run.
#include "../../include/seedpack_amd.h"
#include "launch.h"
#include "linear.h"

namespace spa {
namespace lin {
namespace {

constexpr int COLS = 512, PAIRS = 2048, RUN = 1024;

// Column i of a lane's eight: eight in a row where rows lie at 16-byte addresses, else every 64th, so that a wave's
// loads of one number a lane still are runs of memory.
__device__ __forceinline__ int column(int lane, int i, bool wide8) { return wide8 ? 8 * lane + i : lane + 64 * i; }

template <int KIND>
__device__ __forceinline__ void add8(const void* __restrict__ x, int64_t at, int64_t left, bool wide8, float (&s)[8]) {
    // at, left: the lane's first number, and the columns from there on
    float v[8];
    if (wide8 && left >= 8) {
        load_weights<8>(x, KIND, at, v);
    } else {
        // columns beyond the last are read as the last and dropped: no load waits for a branch
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t c = wide8 ? i : 64 * i, in = at + (c < left ? c : left - 1);
            v[i] = KIND == SRC_F32 ? static_cast<const float*>(x)[in] : wide(static_cast<const uint16_t*>(x)[in], KIND);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (wide8 ? i : 64 * i) < left ? v[i] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = fmaf(v[i], v[i], s[i]);
}

struct Sq {
    const void* x;
    int64_t ld, rows, cols, run;      // run: rows of a workgroup
    const int32_t* which;             // [rows][each], or null
    int each, experts;
    float* part;                      // [runs][experts][cols]
    uint32_t* hits;                   // [runs][experts]
    float* sums;
    int64_t* counts;
    int64_t runs;
    bool wide8;
};

template <int KIND, bool SPLIT>
__global__ __launch_bounds__(256) void k_squares(const Sq q) {
    __shared__ float join[3][COLS];
    __shared__ int list[PAIRS];
    __shared__ int wsum[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t tiles = (q.cols + COLS - 1) / COLS;
    // one expert after another: those with most rows tend to be the first numbers, and the rows under way lie all over x
    // (an expert of each piece in turn, so that its second reader finds it in the caches: 131 instead of 65 us)
    const int64_t pieces = gridDim.x / q.experts;
    const int e = (int)(blockIdx.x / pieces);
    const int64_t piece = blockIdx.x % pieces, run = piece / tiles, c0 = piece % tiles * COLS + column(lane, 0, q.wide8);
    const int64_t r0 = run * q.run, r1 = tmin(q.rows, r0 + q.run), left = q.cols - c0;
    float s[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    uint32_t hits = 0;
    if constexpr (!SPLIT) {
        if (left > 0) {
            int64_t r = r0 + wave;
            for (; r + 12 < r1; r += 16) {                        // four rows' loads under way at once
#pragma unroll
                for (int u = 0; u < 4; ++u) add8<KIND>(q.x, (r + 4 * u) * q.ld + c0, left, q.wide8, s);
            }
            for (; r < r1; r += 4) add8<KIND>(q.x, r * q.ld + c0, left, q.wide8, s);
        }
    } else {
        // (row, expert) pairs, PAIRS at a time: those of this expert listed in their order, each wave a quarter
        const int64_t p1 = r1 * q.each;
        for (int64_t p0 = r0 * q.each; p0 < p1; p0 += PAIRS) {
            constexpr int N = PAIRS / 256;
            int id[N];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int64_t at = p0 + wave * (PAIRS / 4) + i * 64 + lane;
                id[i] = q.which[tmin(at, p1 - 1)];
                if (at >= p1) id[i] = -1;
            }
            uint64_t mask[N];
            int have = 0;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                mask[i] = __ballot(id[i] == e);
                have += __popcll(mask[i]);
            }
            __syncthreads();
            if (lane == 0) wsum[wave] = have;
            __syncthreads();
            int at = 0, total = 0;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                if (w < wave) at += wsum[w];
                total += wsum[w];
            }
            hits += total;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (id[i] == e) {
                    const int64_t pair = p0 + wave * (PAIRS / 4) + i * 64 + lane;
                    list[at + __popcll(mask[i] & ((1ull << lane) - 1))] = (int)(r0 + (uint32_t)(pair - r0 * q.each) / (uint32_t)q.each);
                }
                at += __popcll(mask[i]);
            }
            __syncthreads();
            if (q.wide8 && left >= 8) {
                for (int i = wave; i < total; i += 32) {          // eight rows' loads under way at once, as they lie
                    u4 raw[8][KIND == SRC_F32 ? 2 : 1];
#pragma unroll
                    for (int u = 0; u < 8; ++u) {
                        const int64_t at = (int64_t)list[tmin(i + 4 * u, total - 1)] * q.ld + c0;
                        const u4* p = KIND == SRC_F32 ? reinterpret_cast<const u4*>(static_cast<const float*>(q.x) + at)
                                                      : reinterpret_cast<const u4*>(static_cast<const uint16_t*>(q.x) + at);
                        raw[u][0] = p[0];
                        if (KIND == SRC_F32) raw[u][KIND == SRC_F32] = p[1];
                    }
#pragma unroll
                    for (int u = 0; u < 8; ++u) {
                        if (i + 4 * u >= total) break;
#pragma unroll
                        for (int c = 0; c < 8; ++c) {
                            const float v = KIND == SRC_F32 ? __uint_as_float(raw[u][(KIND == SRC_F32) * (c >> 2)][c & 3])
                                                            : wide((raw[u][0][c >> 1] >> (16 * (c & 1))) & 0xffffu, KIND);
                            s[c] = fmaf(v, v, s[c]);
                        }
                    }
                }
            } else if (left > 0) {
                for (int i = wave; i < total; i += 4) add8<KIND>(q.x, (int64_t)list[i] * q.ld + c0, left, q.wide8, s);
            }
        }
        if (piece % tiles == 0 && threadIdx.x == 0) {
            if (q.runs == 1) q.counts[e] += hits;
            else q.hits[run * q.experts + e] = hits;
        }
    }
    if (wave) {
#pragma unroll
        for (int i = 0; i < 8; ++i) join[wave - 1][i * 64 + lane] = s[i];
    }
    __syncthreads();
    if (wave == 0) {
        float* out = (q.runs == 1 ? q.sums + e * q.cols : q.part + (run * q.experts + e) * q.cols) + c0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int c = column(lane, i, q.wide8) - column(lane, 0, q.wide8);
            float v = (s[i] + join[0][i * 64 + lane]) + (join[1][i * 64 + lane] + join[2][i * 64 + lane]);
            if (c >= left) continue;
            if (q.runs == 1) v = out[c] + v;                      // nothing to join: straight to the caller's sums
            out[c] = v;
        }
    }
    if (!SPLIT && q.runs == 1 && blockIdx.x == 0 && threadIdx.x == 0) q.counts[0] += q.rows;
}

// 32 sums a workgroup, eight lanes to each: every eighth run in turn, the eight then in their order
__global__ __launch_bounds__(256) void k_squares_join(const Sq q) {
    __shared__ float lds[8][32];
    const int64_t n = (int64_t)q.experts * q.cols, i = blockIdx.x * 32ll + (threadIdx.x & 31);
    const int g = threadIdx.x >> 5;
    float v = 0.f;
    if (i < n) {
#pragma unroll 8
        for (int64_t r = g; r < q.runs; r += 8) v += q.part[r * n + i];
    }
    lds[g][threadIdx.x & 31] = v;
    __syncthreads();
    if (g == 0 && i < n) {
#pragma unroll
        for (int j = 1; j < 8; ++j) v += lds[j][threadIdx.x];
        q.sums[i] += v;
    }
    for (int64_t e = blockIdx.x * 256ll + threadIdx.x; e < q.experts; e += gridDim.x * 256ll) {
        int64_t c = q.which ? 0 : q.rows;
        if (q.which)
            for (int64_t r = 0; r < q.runs; ++r) c += q.hits[r * q.experts + e];
        q.counts[e] += c;
    }
}

// Rows of a run. Whole: enough workgroups to fill the device (about 1024 of them), 16 to 1024 rows each (a lane's sum
// over thousands of rows would lose its last bits: 1200000 x 4096 by 9375 rows were 3.9e-6 off), and one launch for up
// to 128. By expert: 1024, so that an expert which gets most of the rows is still spread over many
// workgroups and a workgroup's search of the numbers is worth its rows (16384 x 4096, 64 unlike experts, two for a
// row: runs of 512 91, of 1024 65, of 2048 72, of 8192 202 us).
int64_t run_rows(int64_t rows, int64_t cols, int64_t experts, bool by_expert) {
    const int64_t tiles = (cols + COLS - 1) / COLS * experts;
    int64_t run = rows < RUN ? rows : RUN;
    if (!by_expert) {
        const int64_t runs = tiles < 1024 ? 1024 / tiles : 1;
        run = (rows + runs - 1) / runs;
        if (run < 16) run = 16;
        if (run > RUN) run = RUN;
        if (rows <= 128) run = rows;
    }
    while (run < rows && (rows + run - 1) / run * tiles > (1 << 24)) run *= 2;
    return run;
}
uint64_t part_bytes(int64_t runs, int64_t cols, int64_t experts) {
    return ((uint64_t)runs * experts * cols * 4 + 255) / 256 * 256;
}

}  // namespace
}  // namespace lin
}  // namespace spa

using namespace spa;
using namespace spa::lin;

extern "C" uint64_t spa_add_squares_work_bytes(int64_t rows, int64_t cols, int64_t experts) {
    if (rows <= 0 || cols <= 0 || experts < 0 || rows > INT32_MAX || cols > INT32_MAX || experts > 65535) return 0;
    const bool by_expert = experts != 0;
    if (!by_expert) experts = 1;
    const int64_t run = run_rows(rows, cols, experts, by_expert), runs = (rows + run - 1) / run;
    if (runs == 1) return 0;
    return part_bytes(runs, cols, experts) + ((uint64_t)runs * experts * 4 + 255) / 256 * 256;
}

extern "C" int spa_add_squares(const void* x, int src_kind, int64_t rows, int64_t cols, int64_t x_stride, const int32_t* which,
                               int64_t each, int64_t experts, float* sums, int64_t* counts, void* work, uint64_t work_bytes,
                               void* stream) {
    if (src_kind < SPA_SRC_BF16 || src_kind > SPA_SRC_F32) return fail(SPA_ERR_TYPE, "spa_add_squares: source kind %d", src_kind);
    if (rows < 0 || cols <= 0 || x_stride < cols || rows > INT32_MAX || cols > INT32_MAX)
        return fail(SPA_ERR_ARG, "spa_add_squares: bad shape %lld x %lld, stride %lld", (long long)rows, (long long)cols, (long long)x_stride);
    if (which ? (experts < 1 || experts > 65535 || each < 1 || (rows && each > INT32_MAX / rows)) : experts != 0)
        return fail(SPA_ERR_ARG, "spa_add_squares: %lld experts, %lld for each row", (long long)experts, (long long)each);
    if (rows == 0) return SPA_OK;
    if (!x || !sums || !counts) return fail(SPA_ERR_ARG, "spa_add_squares: null pointer");
    const uintptr_t unit = src_kind == SPA_SRC_F32 ? 3 : 1;
    if ((reinterpret_cast<uintptr_t>(x) & unit) || (reinterpret_cast<uintptr_t>(which) & 3) || (reinterpret_cast<uintptr_t>(sums) & 3) ||
        (reinterpret_cast<uintptr_t>(counts) & 7))
        return fail(SPA_ERR_ARG, "spa_add_squares: a pointer is not aligned to its elements");
    const uint64_t need = spa_add_squares_work_bytes(rows, cols, experts);
    if (need && (!work || (reinterpret_cast<uintptr_t>(work) & 15) || work_bytes < need))
        return fail(SPA_ERR_ARG, "spa_add_squares: needs a 16-byte aligned workspace of spa_add_squares_work_bytes bytes");
    Sq q{};
    q.x = x;
    q.ld = x_stride;
    q.rows = rows;
    q.cols = cols;
    q.which = which;
    q.each = (int)each;
    q.experts = which ? (int)experts : 1;
    q.run = run_rows(rows, cols, q.experts, which != nullptr);
    q.runs = (rows + q.run - 1) / q.run;
    q.part = (float*)work;
    q.hits = (uint32_t*)((uint8_t*)work + part_bytes(q.runs, cols, q.experts));
    q.sums = sums;
    q.counts = counts;
    const int64_t unit16 = src_kind == SPA_SRC_F32 ? 4 : 8;
    q.wide8 = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && x_stride % unit16 == 0;
    hipStream_t st = (hipStream_t)stream;
    const int64_t tiles = (cols + COLS - 1) / COLS;
    if (tiles * q.runs * q.experts > INT32_MAX) return fail(SPA_ERR_ARG, "spa_add_squares: %lld x %lld is too large", (long long)rows, (long long)cols);
    const dim3 grid((unsigned)(tiles * q.runs * q.experts));
#define SPA_SQUARES(KIND)                                                                                   \
    do {                                                                                                    \
        if (which) hipLaunchKernelGGL((k_squares<KIND, true>), grid, dim3(256), 0, st, q);                  \
        else hipLaunchKernelGGL((k_squares<KIND, false>), grid, dim3(256), 0, st, q);                       \
    } while (0)
    if (src_kind == SPA_SRC_BF16) SPA_SQUARES(SRC_BF16);
    else if (src_kind == SPA_SRC_F16) SPA_SQUARES(SRC_F16);
    else SPA_SQUARES(SRC_F32);
#undef SPA_SQUARES
    SPA_HIP_TRY(hipGetLastError());
    if (q.runs == 1) return SPA_OK;
    const int64_t groups = ((int64_t)q.experts * cols + 31) / 32;
    if (groups > INT32_MAX) return fail(SPA_ERR_ARG, "spa_add_squares: %lld experts x %lld is too large", (long long)q.experts, (long long)cols);
    hipLaunchKernelGGL(k_squares_join, dim3((unsigned)groups), dim3(256), 0, st, q);
    SPA_HIP_TRY(hipGetLastError());
    return SPA_OK;
}
