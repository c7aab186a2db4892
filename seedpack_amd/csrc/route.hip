// Routing to experts: each row's experts from its logits, their weights, the slots (row, place) in the order of their
// experts, and the logits' gradient.
//
// A row's scores are s = softmax(l) or 1 / (1 + e^-l). Its experts are those of the largest keys: the logits
// themselves (both scores rise with them), or, with a bias or groups, s + b in 64 bits, for keys are compared with each
// other: in 32 bits one row in some thousands would have two of its experts' keys rounded across each other.
//
// 16 lanes hold a row of up to 256 experts (64 lanes above), so that a wave takes four rows at once and what the lanes
// tell each other stays within 16 of them. A key carries its expert's number in its low bits (reversed: of equal
// keys the lowest number wins), which makes all keys of a row different: each lane sorts its own few, and the
// row's next expert is the largest of 16 heads, whose lane moves its list up.
#include "../../include/seedpack_amd.h"
#include "lanes.h"
#include "launch.h"

#include <math.h>

#include <type_traits>

namespace spa {
namespace {

constexpr int MOST_EXPERTS = 1024, MOST_EACH = 32, MOST_GROUPS = 64;
enum { SOFTMAX = 0, SIGMOID = 1 };

struct Route {
    const void* logits;
    int64_t rows, stride;
    int experts, score, groups, keep, best, each, renorm;
    const float* bias;
    float scale;
    bool wide;               // rows may be read 16 bytes at a time
    int32_t* which;
    float* weights;
};

template <int KIND> __device__ __forceinline__ float logit_at(const void* p, int64_t i) {
    if constexpr (KIND == SRC_F32) return static_cast<const float*>(p)[i];
    const uint32_t h = static_cast<const uint16_t*>(p)[i];
    if constexpr (KIND == SRC_BF16) return bf16_to_f32(h);
    return (float)__builtin_bit_cast(_Float16, (uint16_t)h);
}

// number j of a lane is expert at(j, lane): V neighbours of each run of V L
template <int L, int V> __device__ __forceinline__ int place(int j, int lane) { return j / V * (V * L) + lane * V + j % V; }

template <int KIND, int PER> constexpr int run_of() {
    const int v = KIND == SRC_F32 ? 4 : 8;
    return PER < v ? PER : v;
}

template <int KIND, int L, int PER>
__device__ __forceinline__ void load_row(const void* logits, int64_t at, int experts, bool wide, int lane, float (&x)[PER]) {
    constexpr int V = run_of<KIND, PER>();
#pragma unroll
    for (int j = 0; j < PER; j += V) {
        const int i = place<L, V>(j, lane);
        if (wide && i + V <= experts) {
            if constexpr (KIND == SRC_F32) {
                typedef float fv __attribute__((ext_vector_type(4)));
                const fv v = *reinterpret_cast<const fv*>(static_cast<const float*>(logits) + at + i);
#pragma unroll
                for (int c = 0; c < V; ++c) x[j + c] = v[c];
            } else {
                typedef uint16_t hv __attribute__((ext_vector_type(V)));
                const hv v = *reinterpret_cast<const hv*>(static_cast<const uint16_t*>(logits) + at + i);
#pragma unroll
                for (int c = 0; c < V; ++c) x[j + c] = KIND == SRC_BF16 ? bf16_to_f32(v[c]) : (float)__builtin_bit_cast(_Float16, (uint16_t)v[c]);
            }
        } else {
#pragma unroll
            for (int c = 0; c < V; ++c) x[j + c] = i + c < experts ? logit_at<KIND>(logits, at + i + c) : -INFINITY;
        }
    }
}

// Keys whose order is that of their numbers, zeros of both signs alike and every NaN above all, with the expert's number
// below. 0: not to be chosen. Keys of 64 bits keep 42 of the mantissa.
__device__ __forceinline__ uint64_t key_of(float l, int i) {
    if (l == -INFINITY) return 0;
    uint32_t u = __float_as_uint(l + 0.f);
    if (l != l) u = 0x7fffffffu;
    u = u >> 31 ? ~u : u | 0x80000000u;
    return (uint64_t)u << 32 | (0xffffffffu - (uint32_t)i);
}
__device__ __forceinline__ uint64_t key_of(double s, int i) {
    if (s == -INFINITY) return 0;
    uint64_t u = (uint64_t)__double_as_longlong(s + 0.0);
    if (s != s) u = 0x7fffffffffffffffull;
    u = u >> 63 ? ~u : u | 0x8000000000000000ull;
    return (u & ~1023ull) | (1023 - i);
}
template <typename K> __device__ __forceinline__ K packed(uint64_t k) {
    // 16-bit logits: 19 bits are all that their numbers have, the expert's take the lowest ten
    if constexpr (sizeof(K) == 4) return k ? ((uint32_t)(k >> 32) & ~1023u) | ((uint32_t)k & 1023u) : 0u;
    return k;
}
template <typename K> __device__ __forceinline__ int expert_of(K k) { return 1023 - (int)(k & 1023); }

// Batcher's odd-even merging network: N numbers, the largest first
template <int N, typename K> __device__ __forceinline__ void sort_down(K (&k)[N]) {
#pragma unroll
    for (int p = 1; p < N; p *= 2)
#pragma unroll
        for (int q = p; q >= 1; q /= 2)
#pragma unroll
            for (int j = q % p; j + q < N; j += 2 * q)
#pragma unroll
                for (int i = 0; i < q; ++i) {
                    if (i + j + q >= N || (i + j) / (2 * p) != (i + j + q) / (2 * p)) continue;
                    const K a = k[i + j], b = k[i + j + q];
                    k[i + j] = a > b ? a : b;
                    k[i + j + q] = a > b ? b : a;
                }
}

// the logarithm of a score, up to a number that all of a row's scores share
__device__ __forceinline__ double log_score(float l, int score) {
    if (score == SOFTMAX) return l;
    return l < 0 ? l - log1p(exp((double)l)) : -log1p(exp(-(double)l));
}
__device__ __forceinline__ double logistic(double l) {
    const double e = exp(-fabs(l)), q = 1 / (1 + e);
    return l < 0 ? e * q : q;
}

template <int KIND, int L, int PER, bool DEEP>
__global__ __launch_bounds__(256) void k_route(const Route a) {
    constexpr int ROWS = 256 / L, V = run_of<KIND, PER>(), HELD = MOST_EACH / L > 1 ? MOST_EACH / L : 1;
    typedef typename std::conditional<DEEP || KIND == SRC_F32, uint64_t, uint32_t>::type K;
    extern __shared__ double shared[];
    const int lane = threadIdx.x % L, slot = threadIdx.x / L;
    const int64_t row = (int64_t)blockIdx.x * ROWS + slot;
    const bool in = row < a.rows;
    const int64_t at = (in ? row : 0) * a.stride;

    float x[PER];
    load_row<KIND, L, PER>(a.logits, at, a.experts, a.wide, lane, x);
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < PER; ++j) top = fmaxf(top, x[j]);
    top = row_max<L>(top);

    K k[PER];
    if constexpr (!DEEP) {
#pragma unroll
        for (int j = 0; j < PER; ++j) k[j] = packed<K>(key_of(x[j], place<L, V>(j, lane)));
    } else {
        double s[PER], sum = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            s[j] = a.score == SOFTMAX ? (x[j] == -INFINITY ? 0 : exp((double)x[j] - top)) : logistic(x[j]);
            sum += s[j];
        }
        if (a.score == SOFTMAX) {
            sum = 1 / row_sum<L>(sum);
#pragma unroll
            for (int j = 0; j < PER; ++j) s[j] *= sum;
        }
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int i = place<L, V>(j, lane);
            if (a.bias) s[j] += i < a.experts ? a.bias[i] : 0.f;
            if (x[j] == -INFINITY) s[j] = -INFINITY;
        }
        uint64_t kept = ~0ull;
        const int per = a.experts / a.groups;
        if (a.groups > 1) {
            // each group by as many lanes as there are for it, its two best keys
            double* const keys = shared + slot * (a.experts + MOST_GROUPS);
            double* const score = keys + a.experts;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const int i = place<L, V>(j, lane);
                if (i < a.experts) keys[i] = s[j] == s[j] ? s[j] : INFINITY;
            }
            __syncthreads();
            int lanes = L;
            while (lanes > 1 && lanes * a.groups > L) lanes >>= 1;
            for (int g0 = 0; g0 < a.groups; g0 += L / lanes) {
                const int g = g0 + lane / lanes;
                double one = -INFINITY, two = -INFINITY;
                if (g < a.groups)
                    for (int i = lane % lanes; i < per; i += lanes) {
                        const double v = keys[g * per + i];
                        two = fmax(two, fmin(one, v));
                        one = fmax(one, v);
                    }
                for (int m = 1; m < lanes; m <<= 1) {
                    const double o = lane_xor(one, m), t = lane_xor(two, m);
                    two = fmax(fmax(two, t), fmin(one, o));
                    one = fmax(one, o);
                }
                if (g < a.groups && lane % lanes == 0) score[g] = a.best == 2 && per > 1 ? one + two : one;
            }
            __syncthreads();
            kept = 0;
            for (int g = lane; g < a.groups; g += L) {
                const double mine = score[g];
                int rank = 0;
                for (int o = 0; o < a.groups; ++o) rank += score[o] > mine || (score[o] == mine && o < g);
                if (rank < a.keep) kept |= 1ull << g;
            }
            kept = over_row<L>(kept, [](uint64_t p, uint64_t q) { return p | q; });
        }
        const uint32_t inverse = ((1u << 20) + per - 1) / per;     // i / per for i < 1024
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int i = place<L, V>(j, lane);
            const bool out = i >= a.experts || (a.groups > 1 && !(kept >> ((i * inverse) >> 20) & 1));
            k[j] = out ? 0 : packed<K>(key_of(s[j], i));
        }
    }
    sort_down(k);

    int mine[HELD];
#pragma unroll
    for (int h = 0; h < HELD; ++h) mine[h] = -1;
    for (int j = 0; j < a.each; ++j) {
        const K best = row_max<L>(k[0]);
        if (best && best == k[0]) {
#pragma unroll
            for (int i = 0; i + 1 < PER; ++i) k[i] = k[i + 1];
            k[PER - 1] = 0;
        }
#pragma unroll
        for (int h = 0; h < HELD; ++h)
            if (j == h * L + lane && best) mine[h] = expert_of(best);
    }

    // weights: the chosen scores' ratios from their logarithms, so that none of them vanishes together
    double v[HELD], most = -INFINITY;
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
        const float l = mine[h] < 0 ? -INFINITY : logit_at<KIND>(a.logits, at + mine[h]);
        if (a.renorm) {
            v[h] = mine[h] < 0 ? -INFINITY : log_score(l, a.score);
            most = v[h] > most || v[h] != v[h] ? v[h] : most;
        } else if (a.score == SIGMOID) {
            v[h] = mine[h] < 0 ? 0 : logistic(l);
        } else {
            v[h] = mine[h] < 0 ? 0 : exp((double)l - top);
        }
    }
    double total = 1;
    if (a.renorm) {
        most = row_max<L>(most);
        double sum = 0;
#pragma unroll
        for (int h = 0; h < HELD; ++h) {
            v[h] = mine[h] < 0 ? 0 : exp(v[h] - most);
            sum += v[h];
        }
        total = row_sum<L>(sum);
    } else if (a.score == SOFTMAX) {
        float sum = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) sum += x[j] == -INFINITY ? 0.f : expf(x[j] - top);
        total = row_sum<L>(sum);
    }
    if (!in) return;
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
        const int j = h * L + lane;
        if (j >= a.each) continue;
        a.which[row * a.each + j] = mine[h];
        a.weights[row * a.each + j] = mine[h] < 0 ? 0.f : (float)(a.scale * v[h] / total);
    }
}

template <int KIND, bool DEEP> int route_kind(const Route& a, hipStream_t st) {
    auto go = [&](auto kernel, int rows) {
        const int64_t groups = (a.rows + rows - 1) / rows;
        const size_t bytes = DEEP && a.groups > 1 ? (size_t)rows * (a.experts + MOST_GROUPS) * 8 : 0;
        hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(256), bytes, st, a);
        SPA_HIP_TRY(hipGetLastError());
        return SPA_OK;
    };
    if (a.experts <= 64) return go(k_route<KIND, 16, 4, DEEP>, 16);
    if (a.experts <= 128) return go(k_route<KIND, 16, 8, DEEP>, 16);
    if (a.experts <= 256) return go(k_route<KIND, 16, 16, DEEP>, 16);
    if (a.experts <= 512) return go(k_route<KIND, 64, 8, DEEP>, 4);
    return go(k_route<KIND, 64, 16, DEEP>, 4);
}
template <int KIND> int route_deep(const Route& a, hipStream_t st) {
    return a.bias || a.groups > 1 ? route_kind<KIND, true>(a, st) : route_kind<KIND, false>(a, st);
}

// ---- slots in the order of their experts ----
//
// A counting sort that keeps the order of equal ones: 64 slots are a wave's, whose lanes of the same expert find each
// other by one ballot for each bit of the number; the first of them counts all. A slot's place is the
// number of slots of lower experts, of its expert in earlier runs, and in its own run below it. Numbers outside
// 0..experts-1 count as `experts`: behind all others.
constexpr int RUN = 512, WAVES = RUN / 64;

struct Order {
    const int32_t* which;
    int slots, experts, bits;
    int32_t *order, *starts;
    uint32_t* counts;        // [tile][experts + 1]: a tile's slots of each expert, then their places
    int tiles;
};

// the lanes that hold `key`, of `bits` bits, among those of the wave with `has`
__device__ __forceinline__ uint64_t alike(int key, bool has, int bits) {
    uint64_t m = __ballot(has);
    for (int b = 0; b < bits; ++b) {
        const bool on = key >> b & 1;
        const uint64_t v = __ballot(on);
        m &= on ? v : ~v;
    }
    return m;
}
__device__ __forceinline__ int key_at(const Order& o, int i) {
    const int e = o.which[i];
    return e >= 0 && e < o.experts ? e : o.experts;
}

// everything in one workgroup: counts[run][expert] in LDS
__global__ __launch_bounds__(1024) void k_order_one(const Order o) {
    extern __shared__ uint32_t count[];
    __shared__ uint32_t wave_sum[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, keys = o.experts + 1;
    const int runs = (o.slots + 63) / 64;
    for (int i = threadIdx.x; i < runs * keys; i += 1024) count[i] = 0;
    __syncthreads();
    for (int r = wave; r < runs; r += 16) {
        const int i = r * 64 + lane;
        const bool has = i < o.slots;
        const int key = has ? key_at(o, i) : 0;
        const uint64_t m = alike(key, has, o.bits);
        if (has && (m & ((1ull << lane) - 1)) == 0) count[r * keys + key] = (uint32_t)__popcll(m);
    }
    __syncthreads();
    // each expert's places, thread by thread: up to two experts each (keys <= 1025)
    uint32_t total[2] = {0, 0};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int e = threadIdx.x * 2 + h;
        if (e < keys)
            for (int r = 0; r < runs; ++r) {
                const uint32_t c = count[r * keys + e];
                count[r * keys + e] = total[h];
                total[h] += c;
            }
    }
    uint32_t before = total[0] + total[1];
    const uint32_t own = before;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const uint32_t t = __shfl_up(before, s);
        if (lane >= s) before += t;
    }
    if (lane == 63) wave_sum[wave] = before;
    __syncthreads();
    uint32_t base = before - own;
    for (int w = 0; w < wave; ++w) base += wave_sum[w];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int e = threadIdx.x * 2 + h;
        if (e < keys) {
            o.starts[e] = (int32_t)base;
            for (int r = 0; r < runs; ++r) count[r * keys + e] += base;
        }
        base += total[h];
    }
    __syncthreads();
    for (int r = wave; r < runs; r += 16) {
        const int i = r * 64 + lane;
        const bool has = i < o.slots;
        const int key = has ? key_at(o, i) : 0;
        const uint64_t m = alike(key, has, o.bits);
        if (has) o.order[count[r * keys + key] + __popcll(m & ((1ull << lane) - 1))] = i;
    }
}

// a tile's slots of each expert
__global__ __launch_bounds__(RUN) void k_order_count(const Order o) {
    extern __shared__ uint32_t count[];
    const int keys = o.experts + 1, lane = threadIdx.x & 63;
    for (int e = threadIdx.x; e < keys; e += RUN) count[e] = 0;
    __syncthreads();
    const int i = blockIdx.x * RUN + threadIdx.x;
    const bool has = i < o.slots;
    const int key = has ? key_at(o, i) : 0;
    const uint64_t m = alike(key, has, o.bits);
    if (has && (m & ((1ull << lane) - 1)) == 0) atomicAdd(&count[key], (uint32_t)__popcll(m));
    __syncthreads();
    for (int e = threadIdx.x; e < keys; e += RUN) o.counts[(int64_t)blockIdx.x * keys + e] = count[e];
}

// each expert's counts as sums of the tiles before, and its total: one workgroup an expert
__global__ __launch_bounds__(256) void k_order_scan(const Order o) {
    __shared__ uint32_t wave_sum[4];
    const int keys = o.experts + 1, e = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t carry = 0;
    for (int t0 = 0; t0 < o.tiles; t0 += 256) {
        const int t = t0 + threadIdx.x;
        const uint32_t own = t < o.tiles ? o.counts[(int64_t)t * keys + e] : 0;
        uint32_t sum = own;
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) {
            const uint32_t v = __shfl_up(sum, s);
            if (lane >= s) sum += v;
        }
        __syncthreads();
        if (lane == 63) wave_sum[wave] = sum;
        __syncthreads();
        uint32_t base = carry;
        for (int w = 0; w < 4; ++w) {
            if (w < wave) base += wave_sum[w];
            carry += wave_sum[w];
        }
        if (t < o.tiles) o.counts[(int64_t)t * keys + e] = base + sum - own;
    }
    if (threadIdx.x == 0) o.counts[(int64_t)o.tiles * keys + e] = carry;
}

__global__ __launch_bounds__(RUN) void k_order_place(const Order o) {
    extern __shared__ uint32_t count[];                          // [WAVES][keys], then [keys]
    __shared__ uint32_t wave_sum[WAVES];
    const int keys = o.experts + 1, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t* const base = count + WAVES * keys;
    for (int e = threadIdx.x; e < WAVES * keys; e += RUN) count[e] = 0;
    // where each expert's slots begin: the totals' sums, up to three experts a thread
    constexpr int PER = (MOST_EXPERTS + 1 + RUN - 1) / RUN;
    uint32_t total[PER], sum = 0;
#pragma unroll
    for (int h = 0; h < PER; ++h) {
        const int e = threadIdx.x * PER + h;
        total[h] = e < keys ? o.counts[(int64_t)o.tiles * keys + e] : 0;
        sum += total[h];
    }
    const uint32_t own = sum;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const uint32_t v = __shfl_up(sum, s);
        if (lane >= s) sum += v;
    }
    if (lane == 63) wave_sum[wave] = sum;
    __syncthreads();
    uint32_t at = sum - own;
    for (int w = 0; w < wave; ++w) at += wave_sum[w];
#pragma unroll
    for (int h = 0; h < PER; ++h) {
        const int e = threadIdx.x * PER + h;
        if (e < keys) {
            base[e] = at + o.counts[(int64_t)blockIdx.x * keys + e];
            if (blockIdx.x == 0) o.starts[e] = (int32_t)at;
        }
        at += total[h];
    }
    const int i = blockIdx.x * RUN + threadIdx.x;
    const bool has = i < o.slots;
    const int key = has ? key_at(o, i) : 0;
    const uint64_t m = alike(key, has, o.bits);
    const int below = __popcll(m & ((1ull << lane) - 1));
    if (has && below == 0) count[wave * keys + key] = (uint32_t)__popcll(m);
    __syncthreads();
    if (has) {
        uint32_t p = base[key] + below;
        for (int w = 0; w < wave; ++w) p += count[w * keys + key];
        o.order[p] = i;
    }
}

// one workgroup while its counts fit into a part of LDS that needs no leave
bool one_block(int64_t slots, int64_t experts) { return (slots + 63) / 64 * (experts + 1) * 4 <= 60 * 1024 && slots <= 4096; }
uint64_t order_bytes(int64_t slots, int64_t experts) {
    return one_block(slots, experts) ? 0 : (uint64_t)((slots + RUN - 1) / RUN + 1) * (experts + 1) * 4;
}

int by_expert(const int32_t* which, int64_t slots, int64_t experts, int32_t* order, int32_t* starts, void* work, hipStream_t st) {
    Order o{};
    o.which = which;
    o.slots = (int)slots;
    o.experts = (int)experts;
    while (experts >> o.bits) ++o.bits;
    o.order = order;
    o.starts = starts;
    o.counts = (uint32_t*)work;
    o.tiles = (int)((slots + RUN - 1) / RUN);
    const size_t keys = (size_t)experts + 1;
    if (one_block(slots, experts)) {
        hipLaunchKernelGGL(k_order_one, dim3(1), dim3(1024), (size_t)((slots + 63) / 64) * keys * 4, st, o);
        SPA_HIP_TRY(hipGetLastError());
        return SPA_OK;
    }
    hipLaunchKernelGGL(k_order_count, dim3((unsigned)o.tiles), dim3(RUN), keys * 4, st, o);
    SPA_HIP_TRY(hipGetLastError());
    hipLaunchKernelGGL(k_order_scan, dim3((unsigned)keys), dim3(256), 0, st, o);
    SPA_HIP_TRY(hipGetLastError());
    hipLaunchKernelGGL(k_order_place, dim3((unsigned)o.tiles), dim3(RUN), (WAVES + 1) * keys * 4, st, o);
    SPA_HIP_TRY(hipGetLastError());
    return SPA_OK;
}

// ---- the logits' gradient ----
//
// With a_j = scale w'_j (dw_j - sum_t dw_t w'_t) where the weights were renormalised (w' the chosen scores' shares), else
// scale s_j dw_j:
//   softmax  dl_i = a_i - s_i sum_j a_j     (renormalised: the sum is zero, and no logits but the chosen are read)
//   sigmoid  dl_j = a_j (1 - s_j)
struct Back {
    const void* logits;
    int64_t rows, stride, dstride;
    int experts, score, each, renorm;
    float scale;
    bool wide, dwide;
    const int32_t* which;
    const float* dweights;
    void* dlogits;
};

template <int KIND, int L, int PER>
__global__ __launch_bounds__(256) void k_route_back(const Back a) {
    constexpr int ROWS = 256 / L, V = run_of<KIND, PER>(), HELD = MOST_EACH / L > 1 ? MOST_EACH / L : 1;
    const int lane = threadIdx.x % L;
    const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / L;
    const bool in = row < a.rows;
    const int64_t r = in ? row : 0, at = r * a.stride;

    const bool whole = a.score == SOFTMAX && !a.renorm;
    float p[PER], top = -INFINITY, total = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) p[j] = 0;
    if (whole) {
        load_row<KIND, L, PER>(a.logits, at, a.experts, a.wide, lane, p);
#pragma unroll
        for (int j = 0; j < PER; ++j) top = fmaxf(top, p[j]);
        top = row_max<L>(top);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            p[j] = p[j] == -INFINITY ? 0.f : expf(p[j] - top);
            total += p[j];
        }
        total = row_sum<L>(total);
    }
    int mine[HELD];
    double v[HELD], l[HELD], d[HELD], most = -INFINITY;
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
        const int j = h * L + lane;
        mine[h] = j < a.each ? a.which[r * a.each + j] : -1;
        if (mine[h] >= a.experts) mine[h] = -1;
        l[h] = mine[h] < 0 ? -INFINITY : logit_at<KIND>(a.logits, at + mine[h]);
        d[h] = mine[h] < 0 ? 0 : a.dweights[r * a.each + j];
        if (a.renorm) {
            v[h] = mine[h] < 0 ? -INFINITY : log_score((float)l[h], a.score);
            most = v[h] > most || v[h] != v[h] ? v[h] : most;
        } else if (a.score == SIGMOID) {
            v[h] = mine[h] < 0 ? 0 : logistic(l[h]);
        } else {
            v[h] = mine[h] < 0 ? 0 : exp(l[h] - top) / total;
        }
    }
    if (a.renorm) {
        most = row_max<L>(most);
        double sum = 0, dot = 0;
#pragma unroll
        for (int h = 0; h < HELD; ++h) {
            v[h] = mine[h] < 0 ? 0 : exp(v[h] - most);
            sum += v[h];
            dot += v[h] * d[h];
        }
        sum = row_sum<L>(sum);
        dot = row_sum<L>(dot);
#pragma unroll
        for (int h = 0; h < HELD; ++h) {
            d[h] -= dot / sum;
            v[h] = mine[h] < 0 ? 0 : v[h] / sum;
        }
    }
    float g[HELD];
    double sum = 0;
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
        v[h] = mine[h] < 0 ? 0 : a.scale * v[h] * d[h];
        sum += v[h];
        g[h] = (float)(a.score == SIGMOID && mine[h] >= 0 ? v[h] * logistic(-l[h]) : v[h]);
    }
    if (whole) {
        const float f = (float)(row_sum<L>(sum) / total);
#pragma unroll
        for (int j = 0; j < PER; ++j) p[j] = -p[j] * f;
    }
    const int first = (threadIdx.x & 63) - lane;
    for (int j = 0; j < a.each; ++j) {
        float gv = g[0];
        int e = mine[0];
#pragma unroll
        for (int h = 1; h < HELD; ++h)
            if (j / L == h) {
                gv = g[h];
                e = mine[h];
            }
        gv = __shfl(gv, first + j % L);
        e = __shfl(e, first + j % L);
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (place<L, V>(i, lane) == e) p[i] += gv;
    }
    if (!in) return;
    const int64_t to = row * a.dstride;
#pragma unroll
    for (int j = 0; j < PER; j += V) {
        const int i = place<L, V>(j, lane);
        if constexpr (KIND == SRC_F32) {
            typedef float fv __attribute__((ext_vector_type(4)));
            float* const y = static_cast<float*>(a.dlogits) + to + i;
            if (a.dwide && i + V <= a.experts) {
                *reinterpret_cast<fv*>(y) = fv{p[j], p[j + 1], p[j + 2], p[j + 3]};
            } else {
#pragma unroll
                for (int c = 0; c < V; ++c)
                    if (i + c < a.experts) y[c] = p[j + c];
            }
        } else {
            typedef uint16_t hv __attribute__((ext_vector_type(V)));
            uint16_t* const y = static_cast<uint16_t*>(a.dlogits) + to + i;
            hv w;
#pragma unroll
            for (int c = 0; c < V; ++c)
                w[c] = KIND == SRC_BF16 ? __builtin_bit_cast(uint16_t, (__bf16)p[j + c]) : __builtin_bit_cast(uint16_t, (_Float16)p[j + c]);
            if (a.dwide && i + V <= a.experts) {
                *reinterpret_cast<hv*>(y) = w;
            } else {
#pragma unroll
                for (int c = 0; c < V; ++c)
                    if (i + c < a.experts) y[c] = w[c];
            }
        }
    }
}

template <int KIND> int route_back(const Back& a, hipStream_t st) {
    auto go = [&](auto kernel, int rows) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)((a.rows + rows - 1) / rows)), dim3(256), 0, st, a);
        SPA_HIP_TRY(hipGetLastError());
        return SPA_OK;
    };
    if (a.experts <= 64) return go(k_route_back<KIND, 16, 4>, 16);
    if (a.experts <= 128) return go(k_route_back<KIND, 16, 8>, 16);
    if (a.experts <= 256) return go(k_route_back<KIND, 16, 16>, 16);
    if (a.experts <= 512) return go(k_route_back<KIND, 64, 8>, 4);
    return go(k_route_back<KIND, 64, 16>, 4);
}

bool on(const void* p, uintptr_t unit) { return (reinterpret_cast<uintptr_t>(p) & (unit - 1)) == 0; }

int check_shape(const char* who, int kind, int64_t rows, int64_t experts, int64_t stride, int score, int64_t each) {
    if (kind != SPA_SRC_BF16 && kind != SPA_SRC_F16 && kind != SPA_SRC_F32) return fail(SPA_ERR_TYPE, "%s: logits of kind %d (BF16, F16 and F32 are taken)", who, kind);
    if (score != SOFTMAX && score != SIGMOID) return fail(SPA_ERR_ARG, "%s: unknown score %d", who, score);
    if (experts < 1 || experts > MOST_EXPERTS) return fail(SPA_ERR_ARG, "%s: %lld experts (1 to %d are taken)", who, (long long)experts, MOST_EXPERTS);
    if (each < 1 || each > MOST_EACH || each > experts) return fail(SPA_ERR_ARG, "%s: %lld of %lld experts a row (1 to %d are taken)", who, (long long)each, (long long)experts, MOST_EACH);
    if (rows < 0 || rows * each > INT32_MAX - 1024 || rows > INT32_MAX || stride < experts) return fail(SPA_ERR_ARG, "%s: bad shape %lld x %lld, stride %lld", who, (long long)rows, (long long)experts, (long long)stride);
    return SPA_OK;
}
int check_work(const char* who, const void* work, uint64_t have, uint64_t need) {
    if (need && (!work || !on(work, 256) || have < need))
        return fail(SPA_ERR_ARG, "%s: needs a 256-byte aligned workspace of %llu bytes, got %llu", who, (unsigned long long)need, (unsigned long long)(work ? have : 0));
    return SPA_OK;
}
// runs of V logits at addresses and strides that one load can take
bool wide_rows(const void* p, int kind, int64_t stride) {
    return on(p, 16) && stride % (kind == SPA_SRC_F32 ? 4 : 8) == 0;
}

}  // namespace
}  // namespace spa

using namespace spa;

extern "C" {

uint64_t spa_by_expert_work_bytes(int64_t slots, int64_t experts) {
    if (slots <= 0 || experts < 1 || experts > MOST_EXPERTS) return 0;
    return order_bytes(slots, experts);
}

int spa_by_expert(const int32_t* which, int64_t slots, int64_t experts, int32_t* order, int32_t* starts, void* work,
                  uint64_t work_bytes, void* stream) {
    if (experts < 1 || experts > MOST_EXPERTS) return fail(SPA_ERR_ARG, "by_expert: %lld experts (1 to %d are taken)", (long long)experts, MOST_EXPERTS);
    if (slots < 0 || slots > INT32_MAX - 1024) return fail(SPA_ERR_ARG, "by_expert: %lld slots", (long long)slots);
    if ((slots && (!which || !order)) || !starts) return fail(SPA_ERR_ARG, "by_expert: a pointer is NULL");
    if (int rc = check_work("by_expert", work, work_bytes, spa_by_expert_work_bytes(slots, experts))) return rc;
    return by_expert(which, slots, experts, order, starts, work, (hipStream_t)stream);
}

uint64_t spa_route_work_bytes(int64_t rows, int64_t experts, int64_t each, int sorted) {
    return sorted && rows > 0 && each > 0 ? spa_by_expert_work_bytes(rows * each, experts) : 0;
}

int spa_route(const void* logits, int kind, int64_t rows, int64_t experts, int64_t stride, int score, const float* bias,
              int64_t groups, int64_t keep, int64_t best, int64_t each, int renorm, float scale, int32_t* which,
              float* weights, int32_t* order, int32_t* starts, void* work, uint64_t work_bytes, void* stream) {
    if (int rc = check_shape("route", kind, rows, experts, stride, score, each)) return rc;
    if (groups < 1 || groups > MOST_GROUPS || experts % groups || keep < 1 || keep > groups || (best != 1 && best != 2))
        return fail(SPA_ERR_ARG, "route: %lld of %lld groups of %lld experts by their best %lld (whole groups, up to %d, the best 1 or 2)", (long long)keep, (long long)groups, (long long)experts, (long long)best, MOST_GROUPS);
    if (each > keep * (experts / groups)) return fail(SPA_ERR_ARG, "route: %lld experts a row from %lld groups of %lld", (long long)each, (long long)keep, (long long)(experts / groups));
    if (!order != !starts) return fail(SPA_ERR_ARG, "route: order and starts go together");
    if (rows && (!logits || !which || !weights)) return fail(SPA_ERR_ARG, "route: a pointer is NULL");
    if (int rc = check_work("route", work, work_bytes, spa_route_work_bytes(rows, experts, each, order != nullptr))) return rc;
    hipStream_t st = (hipStream_t)stream;
    if (rows) {
        Route a{logits, rows, stride, (int)experts, score, (int)groups, (int)keep, (int)best, (int)each, renorm, bias, scale, wide_rows(logits, kind, stride), which, weights};
        const int rc = kind == SPA_SRC_BF16 ? route_deep<SRC_BF16>(a, st) : kind == SPA_SRC_F16 ? route_deep<SRC_F16>(a, st) : route_deep<SRC_F32>(a, st);
        if (rc) return rc;
    }
    return order ? by_expert(which, rows * each, experts, order, starts, work, st) : SPA_OK;
}

int spa_route_backward(const void* logits, int kind, int64_t rows, int64_t experts, int64_t stride, int score, int64_t each,
                       int renorm, float scale, const int32_t* which, const float* dweights, void* dlogits, int64_t dstride,
                       void* stream) {
    if (int rc = check_shape("route_backward", kind, rows, experts, stride, score, each)) return rc;
    if (dstride < experts) return fail(SPA_ERR_ARG, "route_backward: rows of %lld at a stride of %lld", (long long)experts, (long long)dstride);
    if (rows && (!logits || !which || !dweights || !dlogits)) return fail(SPA_ERR_ARG, "route_backward: a pointer is NULL");
    if (!rows) return SPA_OK;
    Back a{logits, rows, stride, dstride, (int)experts, score, (int)each, renorm, scale, wide_rows(logits, kind, stride), wide_rows(dlogits, kind, dstride), which, dweights, dlogits};
    hipStream_t st = (hipStream_t)stream;
    return kind == SPA_SRC_BF16 ? route_back<SRC_BF16>(a, st) : kind == SPA_SRC_F16 ? route_back<SRC_F16>(a, st) : route_back<SRC_F32>(a, st);
}

}  // extern "C"
