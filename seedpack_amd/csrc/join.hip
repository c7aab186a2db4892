// The experts' results put together, out[r] = sum_j w[r][j] y[r each + j], and the gradients of both.
//
// Bound by memory: y is read once, 16 bytes a lane.
#include "../../include/seedpack_amd.h"
#include "lanes.h"
#include "launch.h"
#include "linear.h"

namespace spa {
namespace {

struct Join {
    const void *y, *dout;
    int64_t rows, n, ldy, ldo, ldd;
    int64_t first;           // slot of a launch
    int each, experts;
    const float* weights;
    const int32_t* which;    // or NULL: every slot has an expert
    void *out, *dy;
    float* dweights;
    bool wide;
};

template <int KIND> __device__ __forceinline__ float number_at(const void* p, int64_t i) {
    if constexpr (KIND == SRC_F32) return static_cast<const float*>(p)[i];
    const uint32_t h = static_cast<const uint16_t*>(p)[i];
    if constexpr (KIND == SRC_BF16) return bf16_to_f32(h);
    return (float)__builtin_bit_cast(_Float16, (uint16_t)h);
}
template <int KIND> __device__ __forceinline__ void put_number(void* p, int64_t i, float v) {
    if constexpr (KIND == SRC_F32) static_cast<float*>(p)[i] = v;
    else static_cast<uint16_t*>(p)[i] = KIND == SRC_BF16 ? __builtin_bit_cast(uint16_t, (__bf16)v) : __builtin_bit_cast(uint16_t, (_Float16)v);
}
using u4v = lin::u4;
// 16 bytes of numbers as floats, and back
template <int KIND, int V> __device__ __forceinline__ void widen(u4v v, float (&x)[V]) {
#pragma unroll
    for (int c = 0; c < V; ++c) {
        if constexpr (KIND == SRC_F32) x[c] = __uint_as_float(v[c]);
        else {
            const uint32_t h = (v[c >> 1] >> (16 * (c & 1))) & 0xffffu;
            x[c] = KIND == SRC_BF16 ? bf16_to_f32(h) : (float)__builtin_bit_cast(_Float16, (uint16_t)h);
        }
    }
}
template <int KIND, int V> __device__ __forceinline__ u4v shorten(const float (&x)[V]) {
    u4v v = {0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < V; ++c) {
        if constexpr (KIND == SRC_F32) v[c] = __float_as_uint(x[c]);
        else v[c >> 1] |= (uint32_t)(KIND == SRC_BF16 ? __builtin_bit_cast(uint16_t, (__bf16)x[c]) : __builtin_bit_cast(uint16_t, (_Float16)x[c])) << (16 * (c & 1));
    }
    return v;
}
__device__ __forceinline__ bool has_expert(const Join& a, int64_t slot) {
    if (!a.which) return true;
    const int e = a.which[slot];
    return e >= 0 && e < a.experts;
}

// a row's part of up to V numbers; wide: rows begin at whole 16 bytes
template <int KIND, int V> __device__ __forceinline__ void load_part(const void* p, int64_t at, int left, bool wide, float (&x)[V]) {
    if (left >= V) {
        u4v v;
        if constexpr (KIND == SRC_F32) __builtin_memcpy(&v, static_cast<const float*>(p) + at, 16);
        else if (wide) v = *reinterpret_cast<const u4v*>(static_cast<const uint16_t*>(p) + at);
        else v = lin::load8_words(static_cast<const uint16_t*>(p) + at);
        widen<KIND>(v, x);
    } else {
#pragma unroll
        for (int c = 0; c < V; ++c) x[c] = c < left ? number_at<KIND>(p, at + c) : 0.f;
    }
}
template <int KIND, int V> __device__ __forceinline__ void store_part(void* p, int64_t at, int left, const float (&x)[V]) {
    if (left >= V) {
        const u4v v = shorten<KIND>(x);
        __builtin_memcpy(static_cast<char*>(p) + at * (KIND == SRC_F32 ? 4 : 2), &v, 16);    // at any number's address
    } else {
#pragma unroll
        for (int c = 0; c < V; ++c)
            if (c < left) put_number<KIND>(p, at + c, x[c]);
    }
}

template <int KIND>
__global__ __launch_bounds__(256) void k_join(const Join a) {
    constexpr int V = KIND == SRC_F32 ? 4 : 8;
    const int64_t per = (a.n + V - 1) / V, id = blockIdx.x * 256ll + threadIdx.x;
    const int64_t row = id / per, c = (id - row * per) * V;
    if (row >= a.rows) return;
    const int left = (int)(a.n - c < V ? a.n - c : V);
    float sum[V];
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = 0.f;
    for (int j = 0; j < a.each; ++j) {
        const int64_t slot = row * a.each + j;
        if (!has_expert(a, slot)) continue;
        const float w = a.weights[slot];
        float x[V];
        load_part<KIND>(a.y, slot * a.ldy + c, left, a.wide, x);
#pragma unroll
        for (int i = 0; i < V; ++i) sum[i] = fmaf(w, x[i], sum[i]);
    }
    store_part<KIND>(a.out, row * a.ldo + c, left, sum);
}

// One workgroup a slot. A row's slots are of one XCD, which takes every eighth workgroup: dout's row then comes from its L2
// but once (2048 x 4 rows of 4099 in bfloat16: 137 MB read and 36.7 us with the slots in turn, 84 and 29.8 so).
template <int KIND>
__global__ __launch_bounds__(256) void k_join_back(const Join a) {
    constexpr int V = KIND == SRC_F32 ? 4 : 8;
    __shared__ float part[4];
    const uint32_t xcd = blockIdx.x & 7;
    const int64_t slot = a.first + xcd * (gridDim.x / 8) + tmin(xcd, gridDim.x % 8) + (blockIdx.x >> 3), row = slot / a.each;
    const bool has = has_expert(a, slot);
    const float w = has ? a.weights[slot] : 0.f;
    float dot = 0.f;
    for (int64_t c = threadIdx.x * V; c < a.n; c += 256 * V) {
        const int left = (int)(a.n - c < V ? a.n - c : V);
        float d[V], x[V];
        if (has) {
            load_part<KIND>(a.dout, row * a.ldd + c, left, a.wide, d);
            load_part<KIND>(a.y, slot * a.ldy + c, left, a.wide, x);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                dot = fmaf(d[i], x[i], dot);
                d[i] *= w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) d[i] = 0.f;
        }
        store_part<KIND>(a.dy, slot * a.ldo + c, left, d);
    }
    dot = row_sum<64>(dot);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = dot;
    __syncthreads();
    if (threadIdx.x == 0) a.dweights[slot] = (part[0] + part[1]) + (part[2] + part[3]);
}

bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int check(const char* who, int kind, int64_t rows, int64_t each, int64_t n, const int32_t* which, int64_t experts) {
    if (kind != SPA_SRC_BF16 && kind != SPA_SRC_F16 && kind != SPA_SRC_F32) return fail(SPA_ERR_TYPE, "%s: rows of kind %d (BF16, F16 and F32 are taken)", who, kind);
    if (rows < 0 || each < 1 || n < 1 || n > INT32_MAX || rows > INT32_MAX || each > INT32_MAX || rows * each > INT32_MAX - 1024)
        return fail(SPA_ERR_ARG, "%s: bad shape %lld rows of %lld x %lld", who, (long long)rows, (long long)each, (long long)n);
    if (which && (experts < 1 || experts > INT32_MAX)) return fail(SPA_ERR_ARG, "%s: %lld experts", who, (long long)experts);
    return SPA_OK;
}

}  // namespace
}  // namespace spa

using namespace spa;

extern "C" {

int spa_join(const void* y, int kind, int64_t rows, int64_t each, int64_t n, int64_t y_stride, const float* weights,
             const int32_t* which, int64_t experts, void* out, int64_t out_stride, void* stream) {
    if (int rc = check("join", kind, rows, each, n, which, experts)) return rc;
    if (y_stride < n || out_stride < n) return fail(SPA_ERR_ARG, "join: rows of %lld at strides of %lld and %lld", (long long)n, (long long)y_stride, (long long)out_stride);
    if (rows && (!y || !weights || !out)) return fail(SPA_ERR_ARG, "join: a pointer is NULL");
    if (!rows) return SPA_OK;
    const int v = kind == SPA_SRC_F32 ? 4 : 8;
    Join a{};
    a.y = y;
    a.rows = rows;
    a.n = n;
    a.ldy = y_stride;
    a.ldo = out_stride;
    a.each = (int)each;
    a.experts = (int)experts;
    a.weights = weights;
    a.which = which;
    a.out = out;
    a.wide = on16(y) && y_stride % v == 0;
    const int64_t workgroups = (rows * ((n + v - 1) / v) + 255) / 256;
    if (!one_launch(workgroups, 256)) return fail(SPA_ERR_ARG, "join: %lld rows of %lld are more than one launch takes", (long long)rows, (long long)n);
    const dim3 grid((unsigned)workgroups);
    if (kind == SPA_SRC_BF16) hipLaunchKernelGGL(k_join<SRC_BF16>, grid, dim3(256), 0, (hipStream_t)stream, a);
    else if (kind == SPA_SRC_F16) hipLaunchKernelGGL(k_join<SRC_F16>, grid, dim3(256), 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL(k_join<SRC_F32>, grid, dim3(256), 0, (hipStream_t)stream, a);
    SPA_HIP_TRY(hipGetLastError());
    return SPA_OK;
}

int spa_join_backward(const void* y, int kind, int64_t rows, int64_t each, int64_t n, int64_t y_stride, const float* weights,
                      const int32_t* which, int64_t experts, const void* dout, int64_t dout_stride, void* dy,
                      int64_t dy_stride, float* dweights, void* stream) {
    if (int rc = check("join_backward", kind, rows, each, n, which, experts)) return rc;
    if (y_stride < n || dout_stride < n || dy_stride < n) return fail(SPA_ERR_ARG, "join_backward: rows of %lld at strides of %lld, %lld and %lld", (long long)n, (long long)y_stride, (long long)dout_stride, (long long)dy_stride);
    if (rows && (!y || !weights || !dout || !dy || !dweights)) return fail(SPA_ERR_ARG, "join_backward: a pointer is NULL");
    if (!rows) return SPA_OK;
    const int v = kind == SPA_SRC_F32 ? 4 : 8;
    Join a{};
    a.y = y;
    a.dout = dout;
    a.rows = rows;
    a.n = n;
    a.ldy = y_stride;
    a.ldo = dy_stride;
    a.ldd = dout_stride;
    a.each = (int)each;
    a.experts = (int)experts;
    a.weights = weights;
    a.which = which;
    a.dy = dy;
    a.dweights = dweights;
    a.wide = on16(y) && on16(dout) && y_stride % v == 0 && dout_stride % v == 0;
    // a launch takes fewer slots than there may be
    constexpr int64_t PART = 1 << 23;
    static_assert(PART <= UINT32_MAX / 256, "one launch");
    for (a.first = 0; a.first < rows * each; a.first += PART) {
        const int64_t left = rows * each - a.first;
        const dim3 grid((unsigned)(left < PART ? left : PART));
        if (kind == SPA_SRC_BF16) hipLaunchKernelGGL(k_join_back<SRC_BF16>, grid, dim3(256), 0, (hipStream_t)stream, a);
        else if (kind == SPA_SRC_F16) hipLaunchKernelGGL(k_join_back<SRC_F16>, grid, dim3(256), 0, (hipStream_t)stream, a);
        else hipLaunchKernelGGL(k_join_back<SRC_F32>, grid, dim3(256), 0, (hipStream_t)stream, a);
        SPA_HIP_TRY(hipGetLastError());
    }
    return SPA_OK;
}

}  // extern "C"
