// Routing to experts: each row's experts from its logits, their weights, the slots (row, place) in the order of their
// experts, and the logits' gradient.
//
// A row's scores are s = softmax(l) or 1 / (1 + e^-l). Its experts are those of the largest keys: the logits
// themselves (both scores rise with them), or, with a bias or groups, s + b in 64 bits, for keys are compared with each
// other: in 32 bits one row in some thousands would have two of its experts' keys rounded across each other.
//
// A row's lanes, 16, 32 or 64, hold its experts. A key carries its expert's number in its low bits (reversed: of equal
// keys the lowest number wins), which makes all keys of a row different: each lane sorts its own few, and the
// row's next expert is the largest of the lanes' heads, whose lane moves its list up.
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
                typedef float fv __attribute__((ext_vector_type(V)));
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
// below. 0: not to be chosen. Keys of 64 bits keep 42 of the mantissa's bits.
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

// e^x for x <= 0 (NaN stays): x = n ln 2 + r with ln 2 in two parts, and the series to r^13 / 13!, |r| <= 0.347: 4e-18.
// (The library's exp and a division of full rounding, whose arguments may be anything, made 8191 rows of 256 experts
// in groups 19 us.)
__device__ __forceinline__ double exp_down(double x) {
    const double c = fmax(x, -800.), n = rint(c * 1.4426950408889634);
    const double r = fma(n, -0x1.abc9e3b39803fp-56, fma(n, -0x1.62e42fefa39efp-1, c));
    double p = 1. / 6227020800.;
    p = fma(p, r, 1. / 479001600.);
    p = fma(p, r, 1. / 39916800.);
    p = fma(p, r, 1. / 3628800.);
    p = fma(p, r, 1. / 362880.);
    p = fma(p, r, 1. / 40320.);
    p = fma(p, r, 1. / 5040.);
    p = fma(p, r, 1. / 720.);
    p = fma(p, r, 1. / 120.);
    p = fma(p, r, 1. / 24.);
    p = fma(p, r, 1. / 6.);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.);
    p = fma(p, r, 1.);
    p = ldexp(p, (int)n);
    return x == x ? p : x;
}
// 1 / y of 1 <= y <= 2: the hardware's estimate and two steps of Newton's
__device__ __forceinline__ double reciprocal(double y) {
    double r = __builtin_amdgcn_rcp(y);
    r = fma(r, fma(-y, r, 1.), r);
    return fma(r, fma(-y, r, 1.), r);
}
__device__ __forceinline__ double logistic(double l) {
    const double e = exp_down(-fabs(l)), q = reciprocal(1 + e);
    return l < 0 ? e * q : q;
}

// The chosen scores up to a factor that a row's have in common, and their sum. Logistic scores that all but vanish are taken
// by their logarithms: their ratios do not.
template <int L, int HELD>
__device__ __forceinline__ double chosen(const float (&l)[HELD], const int (&mine)[HELD], int score, double (&v)[HELD]) {
    double sum = 0;
    if (score == SIGMOID) {
#pragma unroll
        for (int h = 0; h < HELD; ++h) {
            v[h] = mine[h] < 0 ? 0 : logistic(l[h]);
            sum += v[h];
        }
        sum = row_sum<L>(sum);
        if (!(sum < 1e-280)) return sum;
    }
    // below -600 the logarithm of the logistic is the logit itself
    float most = -INFINITY;
#pragma unroll
    for (int h = 0; h < HELD; ++h) most = mine[h] >= 0 ? fmaxf(most, l[h]) : most;
    most = row_max<L>(most);
    sum = 0;
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
        v[h] = mine[h] < 0 ? 0 : exp_down((double)l[h] - most);
        sum += v[h];
    }
    return row_sum<L>(sum);
}

// what is written to LDS by this wave may be read by it
__device__ __forceinline__ void own_lds() {
    __builtin_amdgcn_wave_barrier();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
}

// numbers of LDS of a row's keys in groups: a group's and a row's begin a bank further than the last one's, for the lanes read
// those of different groups and rows at a time
__host__ __device__ __forceinline__ int group_keys(int experts, int groups) { return (experts + 2 * groups) | 1; }

// One row by its L lanes; keys: LDS for group_keys numbers of its own (DEEP, groups). Lane j of them gives the expert of place
// j + h L in mine[h].
template <int KIND, int L, int PER, bool DEEP, int HELD>
__device__ __forceinline__ void route_row(const Route& a, int64_t row, bool in, int lane, double* keys, int (&mine)[HELD]) {
    constexpr int V = run_of<KIND, PER>();
    typedef typename std::conditional<DEEP || KIND == SRC_F32, uint64_t, uint32_t>::type K;
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
            s[j] = a.score == SOFTMAX ? (x[j] == -INFINITY ? 0 : exp_down((double)x[j] - top)) : logistic(x[j]);
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
        const uint32_t inverse = ((1u << 20) + per - 1) / per;     // i / per for i < 1024
        if (a.groups > 1) {
            // each group by as many lanes as there are for it, its two best keys
            double* const score = keys + a.experts + a.groups;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const int i = place<L, V>(j, lane);
                if (i < a.experts) keys[i + ((i * inverse) >> 20)] = s[j] == s[j] ? s[j] : INFINITY;
            }
            own_lds();
            int lanes = L;
            while (lanes > 1 && lanes * a.groups > L) lanes >>= 1;
            for (int g0 = 0; g0 < a.groups; g0 += L / lanes) {
                const int g = g0 + lane / lanes;
                double one = -INFINITY, two = -INFINITY;
                if (g < a.groups)
                    for (int i = lane % lanes; i < per; i += lanes) {
                        const double v = keys[g * (per + 1) + i];
                        two = fmax(two, fmin(one, v));
                        one = fmax(one, v);
                    }
                for (int m = 1; m < lanes; m <<= 1) {
                    const double o = lane_xor(one, m), t = lane_xor(two, m);
                    two = fmax(fmax(two, t), fmin(one, o));
                    one = fmax(one, o);
                }
                if (g < a.groups && lane % lanes == 0) score[g] = a.best == 2 && per > 1 && one < INFINITY ? one + two : one;   // no inf - inf
            }
            own_lds();
            kept = 0;
            for (int g = lane; g < a.groups; g += L) {
                const double mine = score[g];
                int rank = 0;
                for (int o = 0; o < a.groups; ++o) rank += score[o] > mine || (score[o] == mine && o < g);
                if (rank < a.keep) kept |= 1ull << g;
            }
            kept = over_row<L>(kept, [](uint64_t p, uint64_t q) { return p | q; });
        }
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int i = place<L, V>(j, lane);
            const bool out = i >= a.experts || (a.groups > 1 && !(kept >> ((i * inverse) >> 20) & 1));
            k[j] = out ? 0 : packed<K>(key_of(s[j], i));
        }
    }
    sort_down(k);

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

    float l[HELD];
    double v[HELD], total = 1;
#pragma unroll
    for (int h = 0; h < HELD; ++h) l[h] = mine[h] < 0 ? -INFINITY : logit_at<KIND>(a.logits, at + mine[h]);
    if (a.renorm) {
        total = chosen<L>(l, mine, a.score, v);
    } else {
#pragma unroll
        for (int h = 0; h < HELD; ++h) v[h] = mine[h] < 0 ? 0 : a.score == SIGMOID ? logistic(l[h]) : exp_down((double)l[h] - top);
        if (a.score == SOFTMAX) {
            float sum = 0;
#pragma unroll
            for (int j = 0; j < PER; ++j) sum += x[j] == -INFINITY ? 0.f : expf(x[j] - top);
            total = row_sum<L>(sum);
        }
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

// ---- slots in the order of their experts ----
//
// A counting sort that keeps the order of equal ones. 64 slots are a wave's, whose lanes of the same expert find each
// other by one ballot for each bit of the number; the first of them counts all. A slot's place is the number of slots of
// lower experts, of its expert in earlier tiles, in earlier runs of 64 of its tile, and in its own run below it. Numbers outside
// 0..experts-1 count as `experts`: behind all others.
//
// The routing kernel counts its own rows' experts, a launch adds the counts up, one workgroup an expert, and the last places
// some of the counted tiles at a time; a few rows are routed and ordered by one workgroup, in one launch. (Placing
// workgroups that add up all counts themselves, for one launch less, took 13.5 us for 256 tiles of 128 experts, not 3 and 5.8.)
constexpr int TILE = 512;                // slots that a workgroup places, unless the routing's tiles are larger
constexpr int FEW = 2048;                // slots that one workgroup routes and orders

struct Order {
    const int32_t* which;
    int slots, experts, bits;
    int32_t *order, *starts;
    uint16_t* counts;        // [tiles][experts + 1]: a tile's slots of each expert
    uint32_t* sums;          // [tiles + 1][experts + 1]: those of the tiles before, and all
    int tile, tiles, group;  // slots of a tile, tiles, and the tiles that a workgroup places
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
__device__ __forceinline__ int key_of_slot(const Order& o, int e) { return e >= 0 && e < o.experts ? e : o.experts; }

// inclusive sums over the workgroup's threads; scratch: one number a wave
__device__ __forceinline__ uint32_t running(uint32_t v, uint32_t* scratch) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const uint32_t t = __shfl_up(v, s);
        if (lane >= s) v += t;
    }
    if (lane == 63) scratch[wave] = v;
    __syncthreads();
    for (int w = 0; w < wave; ++w) v += scratch[w];
    return v;
}

constexpr size_t order_lds(int64_t slots, int64_t experts) { return (size_t)((slots + 63) / 64 * 2 + 8) * (experts + 1); }
static_assert(order_lds(TILE, MOST_EXPERTS) <= 64 * 1024, "a tile is placed in the LDS of any launch");

// Places the slots first .. first + n - 1 of `which` (in LDS or memory, from `first` on) by a workgroup of T threads; tile: its
// number. LDS: order_lds(n, experts) bytes, 16-byte aligned.
template <int T>
__device__ __forceinline__ void place_tile(const Order& o, int tile, int first, int n, const int32_t* which, uint8_t* lds) {
    __shared__ uint32_t scratch[T / 64];
    constexpr int PER = (MOST_EXPERTS + T) / T;                  // experts of a thread
    const int keys = o.experts + 1, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, runs = (n + 63) / 64;
    uint32_t *const before = reinterpret_cast<uint32_t*>(lds), *const total = before + keys;
    uint16_t* const count = reinterpret_cast<uint16_t*>(total + keys);
    for (int i = threadIdx.x; i < runs * keys; i += T) count[i] = 0;
    for (int i = threadIdx.x; i < 2 * keys; i += T) before[i] = 0;
    __syncthreads();
    if (o.tiles > 1) {
        for (int e = threadIdx.x; e < keys; e += T) {
            before[e] = o.sums[(int64_t)tile * keys + e];
            total[e] = o.sums[(int64_t)o.tiles * keys + e];
        }
    }
    for (int r = wave; r < runs; r += T / 64) {
        const int i = r * 64 + lane;
        const bool has = i < n;
        const int key = has ? key_of_slot(o, which[i]) : 0;
        const uint64_t m = alike(key, has, o.bits);
        if (has && (m & ((1ull << lane) - 1)) == 0) count[r * keys + key] = (uint16_t)__popcll(m);
    }
    __syncthreads();
    // each expert's runs; then the experts
    uint32_t sum = 0;
#pragma unroll
    for (int h = 0; h < PER; ++h) {
        const int e = threadIdx.x * PER + h;
        if (e < keys) {
            uint32_t c = 0;
            for (int r = 0; r < runs; ++r) {
                const uint32_t v = count[r * keys + e];
                count[r * keys + e] = (uint16_t)c;
                c += v;
            }
            if (o.tiles == 1) total[e] = c;
            sum += total[e];
        }
    }
    uint32_t at = running(sum, scratch) - sum;
#pragma unroll
    for (int h = 0; h < PER; ++h) {
        const int e = threadIdx.x * PER + h;
        if (e < keys) {
            if (tile == 0) o.starts[e] = (int32_t)at;
            before[e] += at;
            at += total[e];
        }
    }
    __syncthreads();
    for (int r = wave; r < runs; r += T / 64) {
        const int i = r * 64 + lane;
        const bool has = i < n;
        const int key = has ? key_of_slot(o, which[i]) : 0;
        const uint64_t m = alike(key, has, o.bits);
        if (has) o.order[before[key] + count[r * keys + key] + __popcll(m & ((1ull << lane) - 1))] = first + i;
    }
}

__global__ __launch_bounds__(512) void k_place(const Order o) {
    extern __shared__ __align__(16) uint8_t lds[];
    const int tile = blockIdx.x * o.group, first = tile * o.tile;
    place_tile<512>(o, tile, first, tmin(o.tile * o.group, o.slots - first), o.which + first, lds);
}

// a tile's slots of each expert
__global__ __launch_bounds__(1024) void k_count(const Order o) {
    extern __shared__ __align__(16) uint8_t lds[];
    uint32_t* const count = reinterpret_cast<uint32_t*>(lds);
    const int keys = o.experts + 1, lane = threadIdx.x & 63;
    for (int e = threadIdx.x; e < keys; e += 1024) count[e] = 0;
    __syncthreads();
    const int first = blockIdx.x * o.tile, n = tmin(o.tile, o.slots - first);
    for (int i0 = 0; i0 < n; i0 += 1024) {
        const int i = i0 + threadIdx.x;
        const bool has = i < n;
        const int key = has ? key_of_slot(o, o.which[first + i]) : 0;
        const uint64_t m = alike(key, has, o.bits);
        if (has && (m & ((1ull << lane) - 1)) == 0) atomicAdd(&count[key], (uint32_t)__popcll(m));
    }
    __syncthreads();
    for (int e = threadIdx.x; e < keys; e += 1024) o.counts[(int64_t)blockIdx.x * keys + e] = (uint16_t)count[e];
}

// each expert's counts added up over the tiles: one workgroup an expert
__global__ __launch_bounds__(256) void k_sums(const Order o) {
    __shared__ uint32_t scratch[4], all;
    const int keys = o.experts + 1, e = blockIdx.x;
    uint32_t carry = 0;
    for (int t0 = 0; t0 < o.tiles; t0 += 256) {
        const int t = t0 + threadIdx.x;
        const uint32_t own = t < o.tiles ? o.counts[(int64_t)t * keys + e] : 0;
        const uint32_t sum = running(own, scratch);
        if (threadIdx.x == 255) all = sum;
        if (t < o.tiles) o.sums[(int64_t)t * keys + e] = carry + sum - own;
        __syncthreads();
        carry += all;
        __syncthreads();
    }
    if (threadIdx.x == 0) o.sums[(int64_t)o.tiles * keys + e] = carry;
}

// the tiles of an order, and its workspace; one tile has no counts, and no byte of `work` is its
void lay_out(Order& o, int64_t slots, int64_t experts, int64_t tile, void* work) {
    o.slots = (int)slots;
    o.experts = (int)experts;
    while (experts >> o.bits) ++o.bits;
    o.tile = (int)tile;
    o.tiles = (int)((slots + tile - 1) / tile);
    o.group = (int)(TILE / tile);
    if (!o.group) o.group = 1;
    if (o.tiles <= 1) return;
    o.counts = static_cast<uint16_t*>(work);
    o.sums = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(work) + ((int64_t)o.tiles * (experts + 1) * 2 + 255) / 256 * 256);
}
uint64_t order_bytes(int64_t slots, int64_t experts, int64_t tile) {
    const int64_t tiles = (slots + tile - 1) / tile, counts = tiles * (experts + 1);
    return tiles > 1 ? (uint64_t)((counts * 2 + 255) / 256 * 256 + (counts + experts + 1) * 4) : 0;
}
// after the counts
int place(const Order& o, hipStream_t st) {
    if (o.tiles > 1) {
        hipLaunchKernelGGL(k_sums, dim3((unsigned)o.experts + 1), dim3(256), 0, st, o);
        SPA_HIP_TRY(hipGetLastError());
    }
    const int64_t most = (int64_t)o.tile * o.group, groups = o.tiles ? ((int64_t)o.tiles + o.group - 1) / o.group : 1;
    hipLaunchKernelGGL(k_place, dim3((unsigned)groups), dim3(512), order_lds(o.slots < most ? o.slots : most, o.experts), st, o);
    SPA_HIP_TRY(hipGetLastError());
    return SPA_OK;
}

int by_expert(const int32_t* which, int64_t slots, int64_t experts, int32_t* order, int32_t* starts, void* work, hipStream_t st) {
    Order o{};
    o.which = which;
    o.order = order;
    o.starts = starts;
    lay_out(o, slots, experts, TILE, work);
    if (o.tiles > 1) {
        hipLaunchKernelGGL(k_count, dim3((unsigned)o.tiles), dim3(1024), (size_t)(experts + 1) * 4, st, o);
        SPA_HIP_TRY(hipGetLastError());
    }
    return place(o, st);
}

// ---- the routing's kernels ----

// Rows by workgroups of 512 (1024 where their registers allow it), `reps` times as many as they hold at once; with counts, the
// slots of each expert among them
template <int KIND, int L, int PER, bool DEEP, int T>
__global__ __launch_bounds__(T) void k_route(const Route a, const Order o, int reps) {
    constexpr int ROWS = T / L, HELD = MOST_EACH / L > 1 ? MOST_EACH / L : 1;
    extern __shared__ __align__(16) uint8_t lds[];
    uint32_t* const count = reinterpret_cast<uint32_t*>(lds);
    const int lane = threadIdx.x % L, slot = threadIdx.x / L, keys = o.experts + 1;
    double* const mine_lds = reinterpret_cast<double*>(lds + (o.counts ? (keys * 4 + 15) / 16 * 16 : 0)) + slot * group_keys(a.experts, a.groups);
    if (o.counts) {
        for (int e = threadIdx.x; e < keys; e += T) count[e] = 0;
        __syncthreads();
    }
    for (int q = 0; q < reps; ++q) {
        const int64_t row = ((int64_t)blockIdx.x * reps + q) * ROWS + slot;
        const bool in = row < a.rows;
        int mine[HELD];
        route_row<KIND, L, PER, DEEP, HELD>(a, row, in, lane, mine_lds, mine);
        if (in && o.counts) {
#pragma unroll
            for (int h = 0; h < HELD; ++h)
                if (h * L + lane < a.each) atomicAdd(&count[mine[h] < 0 ? a.experts : mine[h]], 1u);
        }
    }
    if (o.counts) {
        __syncthreads();
        for (int e = threadIdx.x; e < keys; e += T) o.counts[(int64_t)blockIdx.x * keys + e] = (uint16_t)count[e];
    }
}

// a few rows, a wave each at a time, routed and ordered
template <int KIND, int PER, bool DEEP>
__global__ __launch_bounds__(1024) void k_route_few(const Route a, const Order o) {
    extern __shared__ __align__(16) uint8_t lds[];
    __shared__ int32_t which[FEW];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int row = wave; row < a.rows; row += 16) {
        int mine[1];
        route_row<KIND, 64, PER, DEEP, 1>(a, row, true, lane, reinterpret_cast<double*>(lds) + wave * group_keys(a.experts, a.groups), mine);
        if (lane < a.each) which[row * a.each + lane] = mine[0];
    }
    __syncthreads();
    place_tile<1024>(o, 0, 0, o.slots, which, lds);
}

// How a routing is launched: 64 lanes a row where 16 would leave a long chain of work to few waves (4 rows of 256 experts in
// groups: 13.8 us by 16 lanes), or hold more than 16 numbers each; four times the rows a workgroup of those where there are
// enough, for fewer tiles to add up. Else 16 lanes, or 32 for 129 to 256 experts without bias and groups (8191 rows of 256 in
// float32: 8.8 us; by 64 lanes 14.8); with them 32 lose (21.5 us; by 16 lanes 17.9).
struct Shape {
    bool few;                       // one workgroup does all
    int lanes, threads, rows, reps; // a row's lanes; rows of a workgroup at once, and how often
};
// LDS of a workgroup's rows in groups: 70 KB for 32 rows of 256 experts in 8 groups, 99 KB in 64, of the 160 KB that there are
size_t group_lds(const Route& a, int rows) { return a.groups > 1 ? (size_t)rows * group_keys(a.experts, a.groups) * 8 : 0; }
Shape shape_of(const Route& a, bool deep, bool sorted) {
    Shape s{};
    const int64_t slots = a.rows * a.each;
    s.few = sorted && a.rows <= 64 && slots <= FEW && order_lds(slots, a.experts) <= 50 * 1024 && group_lds(a, 16) <= 50 * 1024;
    s.lanes = a.rows <= 4096 || a.experts > 256 ? 64 : a.experts <= 128 || deep ? 16 : 32;
    s.threads = s.lanes == 16 && !deep ? 1024 : 512;
    s.rows = s.threads / s.lanes;
    s.reps = s.lanes < 64 || a.rows <= 4096 ? 1 : 4;
    return s;
}

template <int KIND, bool DEEP> int route_kind(const Route& a, Order& o, bool sorted, void* work, hipStream_t st) {
    const Shape s = shape_of(a, DEEP, sorted);
    if (s.few) {
        lay_out(o, a.rows * a.each, a.experts, FEW, nullptr);
        size_t bytes = order_lds(o.slots, a.experts);
        if (DEEP && group_lds(a, 16) > bytes) bytes = group_lds(a, 16);
        auto go = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3(1), dim3(1024), bytes, st, a, o);
            SPA_HIP_TRY(hipGetLastError());
            return SPA_OK;
        };
        if (a.experts <= 64) return go(k_route_few<KIND, 1, DEEP>);
        if (a.experts <= 128) return go(k_route_few<KIND, 2, DEEP>);
        if (a.experts <= 256) return go(k_route_few<KIND, 4, DEEP>);
        if (a.experts <= 512) return go(k_route_few<KIND, 8, DEEP>);
        return go(k_route_few<KIND, 16, DEEP>);
    }
    const int64_t rows = (int64_t)s.rows * s.reps, workgroups = (a.rows + rows - 1) / rows;
    if (!one_launch(workgroups, s.threads)) return fail(SPA_ERR_ARG, "route: %lld rows of %d experts are more than one launch takes", (long long)a.rows, a.experts);
    if (sorted) lay_out(o, a.rows * a.each, a.experts, rows * a.each, work);
    const size_t bytes = (sorted ? (size_t)(a.experts + 1 + 3) / 4 * 16 : 0) + (DEEP ? group_lds(a, s.rows) : 0);
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)workgroups), dim3((unsigned)s.threads), bytes, st, a, o, s.reps);
        SPA_HIP_TRY(hipGetLastError());
        return SPA_OK;
    };
    int rc = SPA_OK;
    if (s.lanes == 16) {
        constexpr int T = DEEP ? 512 : 1024;
        if (a.experts <= 64) rc = go(k_route<KIND, 16, 4, DEEP, T>);
        else if (a.experts <= 128) rc = go(k_route<KIND, 16, 8, DEEP, T>);
        else if constexpr (DEEP) rc = go(k_route<KIND, 16, 16, DEEP, T>);
    } else if (s.lanes == 32) {
        if constexpr (!DEEP) rc = go(k_route<KIND, 32, 8, DEEP, 512>);
    } else {
        if (a.experts <= 64) rc = go(k_route<KIND, 64, 1, DEEP, 512>);
        else if (a.experts <= 128) rc = go(k_route<KIND, 64, 2, DEEP, 512>);
        else if (a.experts <= 256) rc = go(k_route<KIND, 64, 4, DEEP, 512>);
        else if (a.experts <= 512) rc = go(k_route<KIND, 64, 8, DEEP, 512>);
        else rc = go(k_route<KIND, 64, 16, DEEP, 512>);
    }
    return rc || !sorted ? rc : place(o, st);
}
template <int KIND> int route_deep(const Route& a, Order& o, bool sorted, void* work, hipStream_t st) {
    return a.bias || a.groups > 1 ? route_kind<KIND, true>(a, o, sorted, work, st) : route_kind<KIND, false>(a, o, sorted, work, st);
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
    float l[HELD];
    double v[HELD], d[HELD];
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
        const int j = h * L + lane;
        mine[h] = j < a.each ? a.which[r * a.each + j] : -1;
        if (mine[h] >= a.experts) mine[h] = -1;
        l[h] = mine[h] < 0 ? -INFINITY : logit_at<KIND>(a.logits, at + mine[h]);
        d[h] = mine[h] < 0 ? 0 : a.dweights[r * a.each + j];
    }
    if (a.renorm) {
        const double sum = chosen<L>(l, mine, a.score, v);
        double dot = 0;
#pragma unroll
        for (int h = 0; h < HELD; ++h) {
            v[h] = mine[h] < 0 ? 0 : v[h] / sum;
            dot += v[h] * d[h];
        }
        dot = row_sum<L>(dot);
#pragma unroll
        for (int h = 0; h < HELD; ++h) d[h] -= dot;
    } else {
#pragma unroll
        for (int h = 0; h < HELD; ++h) v[h] = mine[h] < 0 ? 0 : a.score == SIGMOID ? logistic(l[h]) : exp_down((double)l[h] - top) / total;
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
        sum = row_sum<L>(sum);
        const float f = total == 0.f ? 0.f : (float)(sum / total);   // a row of -inf has no shares
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
        const int64_t workgroups = (a.rows + rows - 1) / rows;
        if (!one_launch(workgroups, 256)) return fail(SPA_ERR_ARG, "route_backward: %lld rows of %d experts are more than one launch takes", (long long)a.rows, a.experts);
        hipLaunchKernelGGL(kernel, dim3((unsigned)workgroups), dim3(256), 0, st, a);
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
    if (rows < 0 || rows > INT32_MAX || rows * each > INT32_MAX - 1024 || stride < experts) return fail(SPA_ERR_ARG, "%s: bad shape %lld x %lld, stride %lld", who, (long long)rows, (long long)experts, (long long)stride);
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
    return order_bytes(slots, experts, TILE);
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
    if (!sorted || rows <= 0 || each <= 0 || each > MOST_EACH || experts < 1 || experts > MOST_EXPERTS) return 0;
    return order_bytes(rows * each, experts, 8 * each);          // the smallest tiles that any form takes
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
    if (!rows) return order ? by_expert(which, 0, experts, order, starts, work, st) : SPA_OK;
    Route a{logits, rows, stride, (int)experts, score, (int)groups, (int)keep, (int)best, (int)each, renorm, bias, scale, wide_rows(logits, kind, stride), which, weights};
    Order o{};
    o.which = which;
    o.order = order;
    o.starts = starts;
    return kind == SPA_SRC_BF16 ? route_deep<SRC_BF16>(a, o, order != nullptr, work, st)
         : kind == SPA_SRC_F16 ? route_deep<SRC_F16>(a, o, order != nullptr, work, st)
                               : route_deep<SRC_F32>(a, o, order != nullptr, work, st);
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
