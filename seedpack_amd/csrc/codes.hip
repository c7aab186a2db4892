// The few-rows product for the block types whose weights are scale x code - offset with small whole codes
// (Q4_0, Q8_0, Q4_K, Q5_K, Q6_K). With w[k] = s c[k] - o over a run of k that shares s and o,
//     sum_k x[k] w[k] = s sum_k x[k] c[k] - o sum_k x[k]:
// the codes, not the weights, are the matrix instruction's operand. A code of up to 7 bits becomes a BF16
// number by putting its bits under the exponent of 128 (0x4300 | c = 128 + c, exact), two codes by one byte
// permutation; 128 s then goes into o. For F16 the same under 1024 (0x6400 | c) and 1024 less, exact too, with what is
// taken from a code of Q4_0, Q6_K or Q8_0: those have no offset then. Nor have Q8_0's beside BF16, signed numbers by
// way of float32. So no weight is rounded, unpacking costs one to one and a half instructions a weight instead of the
// six to eight of decoding to float32 and splitting, and the sums of x alone come from a second instruction with an
// operand of ones, in the registers where they are needed.
//
// The base of 128 costs bits: sums over base + code and less base times the inputs' sum are rounded at 128 scales'
// size, so with codes of half their range a sum's error is that of 5 (Q6_K) to 33 (Q4_0) times as many float32
// roundings, far below a BF16 result's; but a block of a large scale whose codes are all near zero adds errors of its
// scale, not of its weights.
//
// A lane holds 8 codes of weight row lane & 15 for a step of 32 k. A wave works alone on units of 256 k: the
// unit's bytes of its 16 rows go to LDS of its own by 16-byte loads that bypass the registers, each byte
// once (read lane by lane from memory, 32 bytes of a row at a time, the same lines were fetched again and
// again: Q8_0 12288 x 4096 took 63 us, Q6_K 151936 x 1024 149 us), and no barrier is needed before the join. The
// loads of many waves of a compute unit keep the memory busy while others compute.
// Bound by memory latency and, from a few rows on, by the unpacking: one row through two Q4_K matrices 12288 x 4096
// 14.4 us (3.9 TB/s), three through Q6_K 151936 x 1024 31 us (4.1), 32 through Q8_0 12288 x 4096 18.4 us (2.9).
// Q6_K's scales cover 16 k, half a step: its tiles take 8 input rows twice, rows 0-7 with the first 16 k and
// rows 8-15 with the second (zeros elsewhere), so that a lane's sums belong to one scale.
#include "../../include/seedpack_amd.h"
#include "few.h"
#include "launch.h"

namespace spa {
namespace lin {
namespace {

// This lane's row of a unit in LDS: 32-bit words at any byte of it, in pairs that lie 4 bytes on. Words at k and at
// k + 2 (k a multiple of 4) have aligned words and shifts of their own, so that k costs nothing where the caller
// is unrolled. AL: the row begins at a 16-byte address.
template <bool AL>
struct Row {
    const uint32_t* w[2];
    uint32_t sh[2];
    __device__ __forceinline__ void set(const uint8_t* stage, uint32_t mis) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t at = AL ? 0 : mis + 2 * i;
            w[i] = reinterpret_cast<const uint32_t*>(stage) + (at >> 2);
            sh[i] = AL ? 2 * i : at & 3;
        }
    }
    __device__ __forceinline__ u2 pair(int k) const {
        const int i = (k >> 1) & 1;
        const uint32_t* p = w[i] + (k >> 2);
        if (AL && i == 0) return u2{p[0], p[1]};
        const uint32_t a = p[0], b = p[1], c = p[2];
        return u2{__builtin_amdgcn_alignbyte(b, a, sh[i]), __builtin_amdgcn_alignbyte(c, b, sh[i])};
    }
    __device__ __forceinline__ uint32_t word(int k) const {
        const int i = (k >> 1) & 1;
        const uint32_t* p = w[i] + (k >> 2);
        return AL && i == 0 ? p[0] : __builtin_amdgcn_alignbyte(p[1], p[0], sh[i]);
    }
    __device__ __forceinline__ uint32_t half(int k) const {       // k even, two bytes
        if (AL) return (w[0][k >> 2] >> (8 * (k & 2))) & 0xffffu;
        return word(k) & 0xffffu;
    }
};
__device__ __forceinline__ float half_of(uint32_t h) { return (float)__builtin_bit_cast(_Float16, (uint16_t)h); }

typedef _Float16 h2 __attribute__((ext_vector_type(2)));

// codes of up to 8 bits, four bytes -> four numbers: BF16 BASE + code (up to 7 bits), F16 code - LESS
template <int KIND> constexpr float BASE = KIND == SRC_BF16 ? 128.f : 0.f;
template <int KIND, int LESS = 0>
__device__ __forceinline__ void put4(uint32_t c, u4& w, int at) {
    constexpr uint32_t E = KIND == SRC_BF16 ? 0x43434343u : 0x64646464u;
    const uint32_t a = __builtin_amdgcn_perm(E, c, 0x04010400u), b = __builtin_amdgcn_perm(E, c, 0x04030402u);
    constexpr _Float16 TAKEN = 1024 + LESS;
    w[at] = KIND == SRC_BF16 ? a : __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, a) - h2{TAKEN, TAKEN});
    w[at + 1] = KIND == SRC_BF16 ? b : __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, b) - h2{TAKEN, TAKEN});
}

// a unit of 256 weights of one row as lane group g (0..3) reads it; step f: codes 32 f + 8 g .. of it
constexpr int UNIT = 256;
template <int T> struct Unit;

struct K4 {                                                       // Q4_K / Q5_K scales and offsets
    uint32_t sc[2], mn[2];
    float d, dm;
    __device__ __forceinline__ void set(u4 h) {
        d = half_of(h[0] & 0xffffu);
        dm = half_of(h[0] >> 16);
        sc[0] = h[1] & 0x3f3f3f3fu;
        mn[0] = h[2] & 0x3f3f3f3fu;
        sc[1] = (h[3] & 0x0f0f0f0fu) | ((h[1] >> 2) & 0x30303030u);
        mn[1] = ((h[3] >> 4) & 0x0f0f0f0fu) | ((h[2] >> 2) & 0x30303030u);
    }
    template <int KIND> __device__ __forceinline__ void scale(int f, float& s, float& o) const {
        s = d * (float)((sc[f >> 2] >> (8 * (f & 3))) & 0xffu);
        o = fmaf(BASE<KIND>, s, dm * (float)((mn[f >> 2] >> (8 * (f & 3))) & 0xffu));
    }
};
template <> struct Unit<12> {                                     // Q4_K: 4 x 32 bytes of two nibbles
    static constexpr int QK = 256, BS = 144;
    static constexpr bool HALVES = false;
    template <int KIND> static constexpr bool OFFSET = true;
    K4 k;
    template <class R> __device__ __forceinline__ void open(const R& r) { k.set(u4{r.word(0), r.word(4), r.word(8), r.word(12)}); }
    template <int KIND, class R> __device__ __forceinline__ void step(const R& r, int f, int g, u4& w, float& s, float& o) const {
        const u2 q = r.pair(16 + 32 * (f >> 1) + 8 * g);
#pragma unroll
        for (int i = 0; i < 2; ++i) put4<KIND>((f & 1 ? q[i] >> 4 : q[i]) & 0x0f0f0f0fu, w, 2 * i);
        k.scale<KIND>(f, s, o);
    }
};
template <> struct Unit<13> {                                     // Q5_K: the same, and bit f of 32 bytes
    static constexpr int QK = 256, BS = 176;
    static constexpr bool HALVES = false;
    template <int KIND> static constexpr bool OFFSET = true;
    K4 k;
    template <class R> __device__ __forceinline__ void open(const R& r) { k.set(u4{r.word(0), r.word(4), r.word(8), r.word(12)}); }
    template <int KIND, class R> __device__ __forceinline__ void step(const R& r, int f, int g, u4& w, float& s, float& o) const {
        const u2 q = r.pair(48 + 32 * (f >> 1) + 8 * g), h = r.pair(16 + 8 * g);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t lo = (f & 1 ? q[i] >> 4 : q[i]) & 0x0f0f0f0fu;
            put4<KIND>(lo | (((h[i] >> f) & 0x01010101u) << 4), w, 2 * i);
        }
        k.scale<KIND>(f, s, o);
    }
};
template <> struct Unit<14> {                                     // Q6_K: per half of 128, 4 quarters of 32
    static constexpr int QK = 256, BS = 210;
    static constexpr bool HALVES = true;
    template <int KIND> static constexpr bool OFFSET = KIND == SRC_BF16;
    u4 sc;
    float d;
    template <class R> __device__ __forceinline__ void open(const R& r) {
        sc = u4{r.word(192), r.word(196), r.word(200), r.word(204)};
        d = half_of(r.half(208));
    }
    template <int KIND, class R> __device__ __forceinline__ void step(const R& r, int f, int g, u4& w, float& s, float& o) const {
        const int h = f >> 2, qd = f & 3;
        const u2 l = r.pair(64 * h + 32 * (qd & 1) + 8 * g), hi = r.pair(128 + 32 * h + 8 * g);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t c = (qd < 2 ? l[i] : l[i] >> 4) & 0x0f0f0f0fu, b = (hi[i] >> (2 * qd)) & 0x03030303u;
            put4<KIND, 32>(c | (b << 4), w, 2 * i);
        }
        const int byte = (int)(sc[2 * h + (qd >> 1)] << (24 - 16 * (qd & 1) - 8 * (g >> 1))) >> 24;   // scale 8 h + 2 qd + g / 2
        s = d * (float)byte;
        o = OFFSET<KIND> ? (BASE<KIND> + 32.f) * s : 0.f;
    }
};
template <> struct Unit<8> {                                      // Q8_0: blocks of 32 codes of 8 bits
    static constexpr int QK = 32, BS = 34;
    static constexpr bool HALVES = false;
    template <int KIND> static constexpr bool OFFSET = false;
    template <class R> __device__ __forceinline__ void open(const R&) {}
    template <int KIND, class R> __device__ __forceinline__ void step(const R& r, int f, int g, u4& w, float& s, float& o) const {
        const u2 q = r.pair(34 * f + 2 + 8 * g);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (KIND == SRC_F16) {
                put4<KIND, 128>(q[i] ^ 0x80808080u, w, 2 * i);
            } else {
                const float a = (float)(int8_t)q[i], b = (float)(int8_t)(q[i] >> 8), e = (float)(int8_t)(q[i] >> 16), h = (float)((int32_t)q[i] >> 24);
                w[2 * i] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
                w[2 * i + 1] = __builtin_amdgcn_perm(__float_as_uint(h), __float_as_uint(e), 0x07060302u);
            }
        }
        s = half_of(r.half(34 * f));
        o = 0.f;
    }
};
template <> struct Unit<2> {                                      // Q4_0: blocks of 16 low nibbles, then 16 high ones
    static constexpr int QK = 32, BS = 18;
    static constexpr bool HALVES = false;
    template <int KIND> static constexpr bool OFFSET = KIND == SRC_BF16;
    template <class R> __device__ __forceinline__ void open(const R&) {}
    template <int KIND, class R> __device__ __forceinline__ void step(const R& r, int f, int g, u4& w, float& s, float& o) const {
        const u2 q = r.pair(18 * f + 2 + 8 * (g & 1));
#pragma unroll
        for (int i = 0; i < 2; ++i) put4<KIND, 8>((q[i] >> (g & 2 ? 4 : 0)) & 0x0f0f0f0fu, w, 2 * i);
        s = half_of(r.half(18 * f));
        o = OFFSET<KIND> ? (BASE<KIND> + 8.f) * s : 0.f;
    }
};

typedef const __attribute__((address_space(1))) void* gptr;
typedef __attribute__((address_space(3))) void* lptr;

// MT = 1: the inputs are read as they lie, and MR of a lane's four sums count. More tiles: as fragments. AL: every
// unit of a row begins at a 16-byte address.
template <int T, int KIND, int MT, int MR, bool TWO, bool AL, int WAVES>
__global__ __launch_bounds__(WAVES * 64, WAVES < 8 ? 2 : WAVES / 4) void k_codes(const FewArgs a) {
    typedef Unit<T> U;
    constexpr int STEPS = UNIT / 32, AHEAD = MT == 1 ? 8 : (MT == 2 ? 4 : (MT == 4 ? 2 : 1));
    // 16-byte words of a row's unit, wherever in the first of them it begins
    constexpr int BYTES = UNIT / U::QK * U::BS, WORDS = AL ? BYTES / 16 : (BYTES + 15 + 15) / 16, LOADS = (16 * WORDS + 63) / 64;
    constexpr int STAGE = WORDS * 256 + 16, RED = WAVES * (1 + TWO) * MT * 1024, ALL = WAVES * (1 + TWO) * STAGE;
    static_assert(!AL || BYTES % 16 == 0, "units keep the rows' alignment");
    __shared__ __align__(16) uint8_t mem[ALL > RED ? ALL : RED];
    const Few& f = a.f;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n0 = blockIdx.x * 16;
    const int row = lane & 15, g = lane >> 4;
    uint8_t* stage = mem + wave * (1 + TWO) * STAGE;
    // word lane of load i: word c of row r, from the row's first byte on
    uint32_t from[LOADS];
    bool mine[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int word = i * 64 + lane, r = tmin(word / WORDS, 15), c = word % WORDS;
        from[i] = (uint32_t)(tmin(n0 + r, f.n - 1) - n0) * (uint32_t)a.rowbytes + 16 * c;
        mine[i] = word < 16 * WORDS;
    }
    // all words of these rows lie inside the matrix, with those that reach past a unit's end
    const int64_t first = (int64_t)n0 * a.rowbytes, last = (int64_t)tmin(n0 + 16, f.n) * a.rowbytes;
    const bool inside = AL || (first >= 16 && last + 32 <= f.wbytes);
    const uint32_t wrow = (uint32_t)(tmin(n0 + row, f.n - 1) - n0) * (uint32_t)a.rowbytes;
    const int own = U::HALVES ? row & 7 : row;
    const bool live = own < f.m && (!U::HALVES || (row < 8) == (g < 2));
    const uint16_t* xrow = f.x + (live ? own * f.ldx : 0) + 8 * g;
    f4 acc[1 + TWO][MT];
#pragma unroll
    for (int s = 0; s <= TWO; ++s)
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[s][j] = f4{0, 0, 0, 0};
    constexpr uint32_t UNITY = KIND == SRC_BF16 ? 0x3f803f80u : 0x3c003c00u;
    const u4 ones = {UNITY, UNITY, UNITY, UNITY};
    const f4 zero = {0, 0, 0, 0};
    const int units = (f.k + UNIT - 1) / UNIT;
    for (int u = wave; u < units; u += WAVES) {
        const int have = U::QK == UNIT ? STEPS : tmin(STEPS, (f.k - u * UNIT) / 32);
        const int64_t at = first + (int64_t)u * BYTES;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");        // the unit before has been read
#pragma unroll
        for (int h = 0; h <= TWO; ++h) {
            const uint8_t* w = h ? f.w1 : f.w0;
            uint8_t* d = stage + h * STAGE;
            if (inside && have == STEPS) {
#pragma unroll
                for (int i = 0; i < LOADS; ++i) {
                    const uint8_t* p = w + at + from[i];
                    if (!AL) p -= (reinterpret_cast<uintptr_t>(p) & 15);
                    if (mine[i]) __builtin_amdgcn_global_load_lds((gptr)p, (lptr)(d + i * 1024), 16, 0, 0);
                }
            } else {                                              // the matrix's own bytes only
#pragma unroll 1
                for (int i = lane; i < 16 * WORDS; i += 64) {
                    const int r = tmin(n0 + i / WORDS, f.n - 1) - n0;
                    const uint8_t* p = w + at + (int64_t)r * a.rowbytes;
                    p = p - (reinterpret_cast<uintptr_t>(p) & 15) + 16 * (i % WORDS);
                    if (p >= w && p + 16 <= w + f.wbytes) {
                        *reinterpret_cast<u4*>(d + i * 16) = *reinterpret_cast<const u4*>(p);
                        continue;
                    }
#pragma unroll 1
                    for (int k = 0; k < 16; ++k)
                        if (p + k >= w && p + k < w + f.wbytes) d[i * 16 + k] = p[k];
                }
            }
        }
        u4 x0[STEPS];                                             // one tile: all of its unit's inputs on the way too
        if constexpr (MT == 1) {
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                const int k = u * UNIT + 32 * s;
                x0[s] = live && s < have ? *reinterpret_cast<const u4*>(xrow + k) : u4{0, 0, 0, 0};
            }
        }
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        U q[1 + TWO];
        Row<AL> rows[1 + TWO];
#pragma unroll
        for (int h = 0; h <= TWO; ++h) {
            rows[h].set(stage + h * STAGE + row * WORDS * 16, (uint32_t)(reinterpret_cast<uintptr_t>((h ? f.w1 : f.w0) + at + wrow) & 15));
            q[h].open(rows[h]);
        }
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            if (s >= have) break;
            f4 sx[MT];
            u4 x[MT];
#pragma unroll
            for (int j = 0; j < MT; ++j) {
                if constexpr (MT == 1) x[j] = x0[s];
                else x[j] = reinterpret_cast<const u4*>(f.x)[((u * STEPS + s) * MT + j) * 64 + lane];
                if constexpr (U::template OFFSET<KIND>) sx[j] = mul16<KIND>(x[j], ones, zero);
            }
#pragma unroll
            for (int h = 0; h <= TWO; ++h) {
                u4 w;
                float sc, off;
                q[h].template step<KIND>(rows[h], s, g, w, sc, off);
#pragma unroll
                for (int j = 0; j < MT; ++j) {
                    const f4 p = mul16<KIND>(x[j], w, zero);
#pragma unroll
                    for (int c = 0; c < MR; ++c) acc[h][j][c] = fmaf(sc, p[c], U::template OFFSET<KIND> ? fmaf(-off, sx[j][c], acc[h][j][c]) : acc[h][j][c]);
                }
            }
            // no more of x ahead of its use than the registers hold
            if ((s + 1) % AHEAD == 0) asm volatile("" ::: "memory");
        }
    }
    finish<WAVES, MT, TWO, U::HALVES>(f, n0, reinterpret_cast<float*>(mem), acc, Direct<T, U::QK, U::BS>{a, DQ{nullptr}, nullptr});
}

template <int T, int KIND, bool TWO, bool AL>
int launch(const FewArgs& a, hipStream_t st) {
    constexpr int HIGH = Unit<T>::HALVES ? 8 : 16;
    const dim3 grid((unsigned)((a.f.n + 15) / 16));
    const int tiles = few_tiles(T, a.f.m);
    // A wave has at least one unit of k to itself (one row of k = 1024, Q4_K with 4, 8 and 16 waves: n = 4096 7.0, 7.1 and
    // 7.1 us, 12288 6.9, 7.0 and 7.9, 32768 8.4, 10.1 and 17.5, 151936 25, 35 and 71; Q6_K 34, 52 and 85). Few weight rows
    // fill the device with waves only if more of them share a row's k (k = 4096, 8 and 16 waves: n = 4096 Q4_K 6.2 and
    // 6.0, Q8_0 8.1 and 7.5, Q6_K 10.3 and 7.9; 8192 9.0 and 9.7, 11.5 and 12.9, 12.0 and 12.4; 32768 24 and 30, 31 and
    // 42, 32 and 37).
    const int units = (a.f.k + UNIT - 1) / UNIT;
    const bool many = TWO || a.f.n >= 8192, low = units <= 4 && a.f.n >= 4096;
    constexpr int MOST = TWO ? 8 : 16;
#define SPA_CODES(MT, MR, W) hipLaunchKernelGGL((k_codes<T, KIND, MT, MR, TWO, AL, W>), grid, dim3(W * 64), 0, st, a)
#define SPA_CODES_ONE(MR)               \
    do {                                \
        if (low) SPA_CODES(1, MR, 4);   \
        else if (many) SPA_CODES(1, MR, 8); \
        else SPA_CODES(1, MR, MOST);    \
    } while (0)
    if (a.f.m == 1) SPA_CODES_ONE(1);
    else if (tiles == 1) SPA_CODES_ONE(4);
    else if (tiles == 2) SPA_CODES(2, 4, 8);
    else if (tiles == 4) SPA_CODES(4, 4, 8);
    else if constexpr (HIGH == 8) SPA_CODES(8, 4, 8);
#undef SPA_CODES_ONE
#undef SPA_CODES
    SPA_HIP_TRY(hipGetLastError());
    return SPA_OK;
}

template <int T, int KIND, bool TWO>
int aligned(const FewArgs& a, hipStream_t st) {
    if constexpr (UNIT / Unit<T>::QK * Unit<T>::BS % 16 == 0) {
        const uintptr_t at = reinterpret_cast<uintptr_t>(a.f.w0) | reinterpret_cast<uintptr_t>(a.f.w1) | (uintptr_t)a.rowbytes;
        if ((at & 15) == 0) return launch<T, KIND, TWO, true>(a, st);
    }
    return launch<T, KIND, TWO, false>(a, st);
}

template <int T>
int pick(const Few& f, uint16_t* frags, hipStream_t st) {
    FewArgs a{f, f.rowbytes, f.x};
    if (few_tiles(T, f.m) > 1) {
        const int rc = fragments(f, Frags{frags, few_tiles(T, f.m), f.k, Unit<T>::HALVES}, st);
        if (rc) return rc;
        a.f.x = frags;
    }
    if (f.w1) return f.kind == SRC_BF16 ? aligned<T, SRC_BF16, true>(a, st) : aligned<T, SRC_F16, true>(a, st);
    return f.kind == SRC_BF16 ? aligned<T, SRC_BF16, false>(a, st) : aligned<T, SRC_F16, false>(a, st);
}

}  // namespace

int few_codes(const Few& f, uint16_t* frags, hipStream_t st) {
    static_assert(FEW_ROWS == 64, "tiles of up to 64 rows");
    switch (f.type) {
        case 2: return pick<2>(f, frags, st);
        case 8: return pick<8>(f, frags, st);
        case 12: return pick<12>(f, frags, st);
        case 13: return pick<13>(f, frags, st);
        default: return pick<14>(f, frags, st);
    }
}

}  // namespace lin
}  // namespace spa
