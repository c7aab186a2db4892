// The many-rows product of 16-bit operands, sum_k x[m][k] w[n][k], with what follows it in the same
// launch: the adapters' second product, or the gated block's activation and product, or its gradient.
//
// A workgroup computes TN weight rows x TM input rows. Both operands are contiguous along k, so a tile
// step of 64 k is TN + TM rows of 128 bytes; they go from HBM / L2 straight to LDS (16-byte
// buffer loads into LDS) into one of two buffers while the other is multiplied. LDS rows are 128 bytes too,
// their eight 16-byte chunks stored at chunk ^ (row / 2 & 7): a fragment read takes the same chunk of 16
// consecutive rows in a phase, which then lie in 16 different places of the 256 bytes that LDS serves at once
// (with row & 7, which repeats after 8 rows, half of the LDS cycles were conflicts). The exchange is made on
// the global side (a lane fetches the chunk that belongs at its place).
// Weights are the matrix instruction's first operand: a lane then holds four consecutive n of one input
// row, which leave as one 8-byte store.
// For the gated forms half of the TN rows are the gate's and half the same rows of the up projection, so
// that one lane holds both values of an output.
//
// Bound by the matrix unit, whose clock the card's power limit lowers with the data: 4096 x 12288 x 4096 gated in
// BF16 (two products) 658 us, 1250 TFLOP/s, on one card, 695 on another, matrix instructions in 70 to 76 % of the
// cycles; zeros in place of the numbers run a quarter faster. A library's product of one such matrix took 328 us of
// the same data, here 340.
#include "../../include/seedpack_amd.h"
#include "launch.h"
#include "linear.h"

#include <type_traits>

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

typedef __amdgpu_buffer_rsrc_t rsrc;
typedef __attribute__((address_space(3))) void* lptr;
typedef uint16_t h2u __attribute__((ext_vector_type(2)));

// the least adapter number above `after` among the tile's rows (held by the wave's lanes), or INT32_MAX
template <int N>
__device__ __forceinline__ int next_adapter(const int (&ids)[N], int after) {
    int best = INT32_MAX;
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (ids[i] > after) best = tmin(best, ids[i]);
#pragma unroll
    for (int s = 32; s; s >>= 1) best = tmin(best, __shfl_xor(best, s));
    return __builtin_amdgcn_readfirstlane(best);
}

template <int HALF, int TN, int TM, int WN, int WM, int OUT>
__device__ __forceinline__ void product(const Gemm& g) {
    constexpr int NW = WN * WM;                              // waves
    constexpr bool TWO = OUT == OUT_GATED || OUT == OUT_GRAD;
    constexpr int TNE = TWO ? TN / 2 : TN;                   // output columns of the tile
    constexpr int FN = TN / WN / 32, FM = TM / WM / 32;      // 32 x 32 fragments of a wave
    constexpr int LOADS = (TN + TM) / 8 / NW;                // 8 rows by one load of a wave
    static_assert((TN + TM) % (8 * NW) == 0 && (!TWO || FN % 2 == 0), "tile shape");
    // a wave's outputs on their way out: its input rows x its columns, rows 16 bytes apart from a power of two
    constexpr int ROWS = TM / WM, COLS = TN / WN, PITCH = COLS + 8;
    constexpr int STAGES = 2 * (TN + TM) * BK, OUTS = OUT == OUT_PART ? NW * 64 * (COLS + 4) : NW * ROWS * PITCH;
    __shared__ __align__(16) uint16_t mem[STAGES > OUTS ? STAGES : OUTS];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // Tiles are dealt so that each of the 8 XCDs, which take workgroups in turn, has a run of neighbours
    // (its L2 then serves their shared rows) of one piece of k, and a run covers 8 tiles of input rows per tile of weights.
    const int nt = (g.n + TNE - 1) / TNE, mt = (g.m + TM - 1) / TM, total = nt * mt;
    int id, piece = 0, side = 0;
    {
        const int all = gridDim.x, q = all / 8, r = all % 8, xcd = blockIdx.x & 7, at = blockIdx.x >> 3;
        id = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + at;
    }
    const uint16_t* w0 = g.w0;
    int k0 = 0, steps = g.k / BK;
    if (OUT == OUT_PART) {                                        // a piece of k of one matrix
        piece = id / total;
        id -= piece * total;
        side = piece / g.pieces;
        piece -= side * g.pieces;
        if (side) w0 = g.w1;
        k0 = steps * piece / g.pieces;
        steps = steps * (piece + 1) / g.pieces - k0;
    }
    constexpr int GROUP = 8;
    const int band = id / (GROUP * nt), in = id - band * GROUP * nt;
    const int height = tmin(GROUP, mt - band * GROUP);
    const int m0 = (band * GROUP + in % height) * TM, n0 = in / height * TNE;

    if (OUT == OUT_PART && g.which) {                             // a tile that serves none of its rows
        const int a0 = n0 / g.rank, a1 = (tmin(n0 + TNE, g.n) - 1) / g.rank;
        bool any = false;
#pragma unroll
        for (int i = 0; i < TM / 64; ++i) {
            const int a = g.which[tmin(m0 + 64 * i + lane, g.m - 1)];
            any = any || (a >= a0 && a <= a1);
        }
        if (!__ballot(any)) return;                               // the same in every wave
    }

    // where this lane fetches from: row lane / 8 of an 8-row load, the chunk that belongs at its place. Buffer
    // loads, whose addresses are a wave's base and a lane's 32-bit offset (and whose LDS writes, unlike those of
    // global loads, do not make the compiler wait for every LDS read at once).
    uint32_t off[LOADS];
    static_assert(NW % 2 == 0, "the parity of an 8-row load is its wave's");
    const int lr = lane >> 3, chunk = (lane & 7) ^ ((lr >> 1) + 4 * (wave & 1));
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
        const int r0 = (j * NW + wave) * 8;
        if (r0 < TN) off[j] = (uint32_t)(tmin(n0 + r0 - (TWO && r0 >= TNE ? TNE : 0) + lr, g.n - 1) - n0) * (uint32_t)(2 * g.ldw);
        else off[j] = (uint32_t)(tmin(m0 + r0 - TN + lr, g.m - 1) - m0) * (uint32_t)(2 * g.ldx);
        off[j] += 16 * chunk;
    }
    constexpr int RAW = 0x00027000;                               // a plain buffer of bytes
    const rsrc rw0 = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(w0 + (int64_t)n0 * g.ldw + k0 * BK), 0, -1, RAW);
    const rsrc rw1 = TWO ? __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(g.w1 + (int64_t)n0 * g.ldw + k0 * BK), 0, -1, RAW) : rw0;
    const rsrc rx = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(g.x + (int64_t)m0 * g.ldx + k0 * BK), 0, -1, RAW);
    auto fetch = [&](int buf, int kt, int j0, int j1) {
#pragma unroll
        for (int j = j0; j < j1; ++j) {
            // a load of all waves lies in one operand
            static_assert(TNE % (8 * NW) == 0 && TN % (8 * NW) == 0, "tile shape");
            const rsrc r = j * NW * 8 >= TN ? rx : (TWO && j * NW * 8 >= TNE ? rw1 : rw0);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lptr)(mem + buf * (TN + TM) * BK + (j * NW + wave) * 8 * BK), 16, off[j], kt * (2 * BK), 0, 0);
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

    // Fragments are read one part of 16 k ahead of their use. In a tile's last part the other buffer's first
    // fragments are read: before it, every wave's fetches into that buffer have arrived and every wave has read the
    // last of this one, so one barrier a tile orders both, and this buffer's next contents, fetched right after
    // it, have a whole tile's time to arrive.
    constexpr int PARTS = BK / 16;
    u4 fa[2][FN], fb[2][FM];
    auto read = [&](int buf, int part, int to) {
        const uint16_t* t = mem + buf * (TN + TM) * BK;
#pragma unroll
        for (int i = 0; i < FN; ++i)
            fa[to][i] = *reinterpret_cast<const u4*>(t + arow[i] * BK + (((2 * part + fk) ^ ((arow[i] >> 1) & 7)) * 8));
#pragma unroll
        for (int i = 0; i < FM; ++i)
            fb[to][i] = *reinterpret_cast<const u4*>(t + brow[i] * BK + (((2 * part + fk) ^ ((brow[i] >> 1) & 7)) * 8));
    };
    // One tile step; N1, N2: there is a next one, and one after that. Fetches, fragment reads and products are
    // dealt out in turn: a wave whose fetches (eight in a row) or reads queue up would issue no product meanwhile.
    constexpr int EARLY = LOADS / 2;
    auto tile_step = [&](int kt, auto n1, auto n2) {
        constexpr bool N1 = decltype(n1)::value, N2 = decltype(n2)::value;
        const int buf = kt & 1;
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
            const bool last = part == PARTS - 1;
            auto products = [&](int i0, int i1) {
#pragma unroll
                for (int i = i0; i < i1; ++i)
#pragma unroll
                    for (int j = 0; j < FM; ++j) acc[i][j] = Op<HALF>::mul(fa[part & 1][i], fb[part & 1][j], acc[i][j]);
            };
            constexpr int AHEAD = FN / 4 > 0 ? FN / 4 : 1;        // (none: 2 % longer)
            if (last && N1) {
                // some of the part's products are under way while the waves meet
                products(0, AHEAD);
                __builtin_amdgcn_sched_barrier(0);
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            }
            if (!last) read(buf, part + 1, (part + 1) & 1);
            else if (N1) read(buf ^ 1, 0, 0);
            if (part == 0 && N1) fetch(buf ^ 1, kt + 1, EARLY, LOADS);
            if (last && N2) fetch(buf, kt + 2, 0, EARLY);
            products(last && N1 ? AHEAD : 0, FN);
#pragma unroll
            for (int i = 0; i < FN * FM; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x010, 1, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    fetch(0, 0, 0, LOADS);
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    if (steps > 1) fetch(1, 1, 0, EARLY);
    read(0, 0, 0);
    for (int kt = 0; kt < steps - 2; ++kt) tile_step(kt, std::true_type(), std::true_type());
    if (steps > 1) tile_step(steps - 2, std::true_type(), std::false_type());
    tile_step(steps - 1, std::false_type(), std::false_type());

    // Lane: input row (lane & 31) of a fragment; register 4 q + c: weight row 8 q + 4 (lane >> 5) + c. Stored as
    // they lie, a wave would write 16 bytes to each of 32 rows at a time; by way of LDS, which the loop is done with,
    // it writes (and reads dh) in runs of its columns.
    const int nw = n0 + wn * (TNE / WN) + 4 * fk, mw = m0 + wm * ROWS;
    uint16_t* const out = mem + wave * ROWS * PITCH;
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    auto place = [&](int j, int i, int q) -> u2& {
        return *reinterpret_cast<u2*>(out + (32 * j + fr) * PITCH + 32 * i + 8 * q + 4 * fk);
    };
    // columns c0.. of the staged rows to or from columns n.. of a matrix, `most` columns wide, eight numbers a lane
    constexpr int RUN = TNE / WN;
    auto flush = [&](uint16_t* y, int64_t ld, int c0, int most, bool again) {
        const bool wide16 = (ld & 7) == 0 && (reinterpret_cast<uintptr_t>(y) & 15) == 0;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        for (int u = lane; u < ROWS * (RUN / 8); u += 64) {
            const int r = u / (RUN / 8), c = u % (RUN / 8) * 8, n = n0 + wn * RUN + c;
            if (mw + r >= g.m || n >= most) continue;
            uint16_t* p = y + (int64_t)(mw + r) * ld + n;
            u4 v = *reinterpret_cast<const u4*>(out + r * PITCH + c0 + c);
            if (again) v = u4{finite2(v[0]), finite2(v[1]), finite2(v[2]), finite2(v[3])};
            if (wide16 && n + 8 <= most) {
                __builtin_nontemporal_store(v, reinterpret_cast<u4*>(p));
            } else if (n + 8 <= most) {
                __builtin_memcpy(p, &v, 16);                      // at any number's address
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (n + k < most) p[k] = (uint16_t)(v[k >> 1] >> (16 * (k & 1)));
            }
        }
    };
    if constexpr (!TWO) {
        const int32_t* const we = side ? g.we1 : g.we0;
        const bool scaled = g.xe || we;
        bool unscaled = false;
        auto unscale = [&](int i, int j, f16v& v) {
            if (!scaled || unscaled) return;
            const int mi = tmin(m0 + brow[j] - TN, g.m - 1), xe = g.xe ? g.xe[mi] : 0;
#pragma unroll
            for (int c = 0; c < 16; ++c) {
                const int ni = tmin(nw + 32 * i + 8 * (c >> 2) + (c & 3), g.n - 1);
                v[c] = ldexpf(v[c], xe + (we ? we[ni] : 0));
            }
        };
        const Expand& ex = g.ex;
        // pieces of k share the ranks, 16 at a time
        const int first = OUT == OUT_PART ? piece * 16 : 0, stride = OUT == OUT_PART ? g.pieces * 16 : 16;
        bool odd = false;                                         // some number of b was not finite
        if (OUT == OUT_LOW || (OUT == OUT_PART && g.ex.low)) {
            // the adapters' second product, one adapter of the tile's rows at a time: rows of another
            // adapter take part with zeros. low is split into two BF16 parts, b into two where it is F16. An infinity
            // of low is in its second part alone, which meets b's first: b's second may be zero. Infinities and NaN of
            // b, which zeros would make NaN in other adapters' rows, are the largest number here; their rows
            // get them below.
#pragma unroll
            for (int j = 0; j < FM; ++j)
#pragma unroll
                for (int i = 0; i < FN; ++i) unscale(i, j, acc[i][j]);
            unscaled = true;
            int mine[FM], zrow[FM], brow0[FN];
#pragma unroll
            for (int j = 0; j < FM; ++j) {
                const int mi = m0 + brow[j] - TN;
                zrow[j] = tmin(mi, g.m - 1);
                mine[j] = mi < g.m ? ex.which[zrow[j]] : -1;
            }
#pragma unroll
            for (int i = 0; i < FN; ++i) brow0[i] = tmin(n0 + arow[i], g.n - 1);
            // rows and columns beyond the last are read as the last: they are not kept
            int ids[TM / 64];                                     // those outside the pool as -1
#pragma unroll
            for (int i = 0; i < TM / 64; ++i) {
                const int mi = m0 + 64 * i + lane, a = ex.which[tmin(mi, g.m - 1)];
                ids[i] = mi < g.m && a < ex.pool ? a : -1;
            }
            for (int a = next_adapter(ids, -1); a != INT32_MAX; a = next_adapter(ids, a)) {
                const uint16_t* ba = ex.b + (int64_t)a * g.n * ex.rank;
                for (int r0 = first; r0 < ex.rp; r0 += stride) {
                    const int r = r0 + 8 * fk;
                    f4 z[FM][2];
                    u4 h[FN];
#pragma unroll
                    for (int j = 0; j < FM; ++j)
#pragma unroll
                        for (int c = 0; c < 2; ++c) z[j][c] = *reinterpret_cast<const f4*>(ex.low + (int64_t)zrow[j] * ex.rp + r + 4 * c);
#pragma unroll
                    for (int i = 0; i < FN; ++i) {
                        const uint16_t* p = ba + (int64_t)brow0[i] * ex.rank;
                        if (ex.wide_b) {                          // rank a multiple of 8: eight ranks there or none
                            h[i] = *reinterpret_cast<const u4*>(p + tmin(r, ex.rank - 8));
                        } else {
#pragma unroll
                            for (int c = 0; c < 4; ++c) {
                                const uint32_t lo = p[tmin(r + 2 * c, ex.rank - 1)], hi = p[tmin(r + 2 * c + 1, ex.rank - 1)];
                                h[i][c] = lo | (hi << 16);
                            }
                        }
                    }
                    // ranks beyond the last: low holds zeros there, b's numbers are cleared (they may be infinite)
                    h2u largest = {0, 0};
#pragma unroll
                    for (int i = 0; i < FN; ++i)
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const int left = ex.rank - r - 2 * c;
                            h[i][c] &= left >= 2 ? 0xffffffffu : (left == 1 ? 0xffffu : 0u);
                            const uint32_t size = h[i][c] & 0x7fff7fffu;
                            largest = __builtin_elementwise_max(largest, __builtin_bit_cast(h2u, size));
                        }
                    const uint32_t top = ex.kind == SRC_BF16 ? 0x7f80u : 0x7c00u;
                    if (__ballot(largest[0] >= top || largest[1] >= top)) {
                        odd = true;
#pragma unroll
                        for (int i = 0; i < FN; ++i)
#pragma unroll
                            for (int c = 0; c < 4; ++c) {
                                if ((h[i][c] & top) == top) h[i][c] = (h[i][c] & 0xffff8000u) | (top - 1);
                                if ((h[i][c] >> 16 & top) == top) h[i][c] = (h[i][c] & 0x8000ffffu) | (top - 1) << 16;
                            }
                    }
                    bf8 zh[FM], zl[FM];
#pragma unroll
                    for (int j = 0; j < FM; ++j) {
                        float v[8], w[8];
#pragma unroll
                        for (int c = 0; c < 8; ++c) {
                            v[c] = mine[j] == a ? z[j][c >> 2][c & 3] : 0.f;
                            w[c] = __builtin_isinf(v[c]) ? 0.f : v[c];
                        }
                        split8(w, zh[j], zl[j]);
#pragma unroll
                        for (int c = 0; c < 8; ++c)
                            if (__builtin_isinf(v[c])) zl[j][c] = (__bf16)v[c];
                    }
#pragma unroll
                    for (int i = 0; i < FN; ++i) {
                        bf8 bh = __builtin_bit_cast(bf8, h[i]), bl;
                        if (ex.kind != SRC_BF16) {
                            float v[8];
#pragma unroll
                            for (int c = 0; c < 8; ++c) v[c] = wide((h[i][c >> 1] >> (16 * (c & 1))) & 0xffffu, SRC_F16);
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
        // what the numbers of b that are not finite give output (mi, ni): infinities, NaN, or nothing
        auto lost = [&](int mi, int ni) {
            float t = 0.f;
            const int a = ex.which[mi];
            if (a < 0 || a >= ex.pool) return t;
            const uint16_t* p = ex.b + ((int64_t)a * g.n + ni) * ex.rank;
            for (int r0 = first; r0 < ex.rank; r0 += stride)
                for (int r = r0; r < tmin(r0 + 16, ex.rank); ++r) {
                    const float b = wide(p[r], ex.kind);
                    if (!(fabsf(b) <= 3.4028235e38f)) t = fmaf(ex.low[(int64_t)mi * ex.rp + r], b, t);
                }
            return t;
        };
        if constexpr (OUT == OUT_PART) {
            // float32 sums, 32 input rows at a time through the wave's staging place
            float* const stage = reinterpret_cast<float*>(mem) + wave * 32 * (COLS + 4);
            float* const part = g.part + ((int64_t)(side * g.pieces + piece) * g.m) * g.n;
#pragma unroll
            for (int j = 0; j < FM; ++j) {
#pragma unroll
                for (int i = 0; i < FN; ++i) {
                    f16v v = acc[i][j];
                    unscale(i, j, v);
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        *reinterpret_cast<f4*>(stage + fr * (COLS + 4) + 32 * i + 8 * q + 4 * fk) = f4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
                }
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                for (int u = lane; u < 32 * (COLS / 4); u += 64) {
                    const int r = u / (COLS / 4), c = u % (COLS / 4) * 4, n = n0 + wn * COLS + c, mi = mw + 32 * j + r;
                    if (mi >= g.m || n >= g.n) continue;
                    f4 v = *reinterpret_cast<const f4*>(stage + r * (COLS + 4) + c);
                    if (odd)
                        for (int k = 0; k < 4; ++k)
                            if (n + k < g.n) v[k] += lost(mi, n + k);
                    float* p = part + (int64_t)mi * g.n + n;
                    if (n + 4 <= g.n) {
                        __builtin_memcpy(p, &v, 16);              // at any number's address
                    } else {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (n + k < g.n) p[k] = v[k];
                    }
                }
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            }
            return;
        }
#pragma unroll
        for (int j = 0; j < FM; ++j)
#pragma unroll
            for (int i = 0; i < FN; ++i) {
                f16v v = acc[i][j];
                unscale(i, j, v);
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    place(j, i, q) = u2{narrow2(v[4 * q], v[4 * q + 1], g.kind), narrow2(v[4 * q + 2], v[4 * q + 3], g.kind)};
            }
        if (odd) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            for (int u = lane; u < ROWS * COLS; u += 64) {
                const int r = u / COLS, c = u % COLS, n = n0 + wn * COLS + c;
                if (mw + r >= g.m || n >= g.n) continue;
                const float t = lost(mw + r, n);
                uint16_t& at = out[r * PITCH + c];
                if (t != 0.f) at = narrow(wide(at, g.kind) + t, g.kind);
            }
        }
        flush(g.y, g.ldy, 0, g.n, false);
    } else {
        if constexpr (OUT == OUT_GRAD) {                          // dh to where its gate's gradient will lie
            for (int u = lane; u < ROWS * (RUN / 8); u += 64) {
                const int r = u / (RUN / 8), c = u % (RUN / 8) * 8, n = n0 + wn * RUN + c;
                u4 v = {0, 0, 0, 0};
                if (mw + r < g.m && n < g.n) {
                    const uint16_t* p = g.dh + (int64_t)(mw + r) * g.ldh + n;
                    if (n + 8 <= g.n) {
                        __builtin_memcpy(&v, p, 16);
                    } else {
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            if (n + k < g.n) v[k >> 1] |= (uint32_t)p[k] << (16 * (k & 1));
                    }
                }
                *reinterpret_cast<u4*>(out + r * PITCH + c) = v;
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
#pragma unroll
        for (int j = 0; j < FM; ++j) {
            const int mi = tmin(m0 + brow[j] - TN, g.m - 1);
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
                    u2& at = place(j, i, q);
                    if constexpr (OUT == OUT_GATED) {
#pragma unroll
                        for (int c = 0; c < 4; ++c) gv[c] = act_value(gv[c], g.act) * uv[c];
                    } else {
                        const u2 d4 = at;
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            // columns n..np-1 are padding of the products that follow: zeros, whatever the sums are
                            const float d = wide((d4[c >> 1] >> (16 * (c & 1))) & 0xffffu, g.kind);
                            float value, slope;
                            act_both(gv[c], g.act, value, slope);
                            const bool in = ni + c < g.n;
                            gv[c] = in ? ldexpf(d * uv[c] * slope, e0[c] - ge) : 0.f;
                            uv[c] = in ? ldexpf(d * value, e1[c] - ge) : 0.f;
                        }
                        (&at)[RUN / 4] = u2{narrow2(uv[0], uv[1], HALF), narrow2(uv[2], uv[3], HALF)};
                    }
                    const int kind = OUT == OUT_GRAD ? HALF : g.kind;
                    at = u2{narrow2(gv[0], gv[1], kind), narrow2(gv[2], gv[3], kind)};
                }
        }
        if constexpr (OUT == OUT_GATED) {
            flush(g.y, g.ldy, 0, g.n, false);
        } else {
            for (int64_t at = 0; at <= (g.twice ? 2 * g.np : 0); at += 2 * g.np) {
                flush(g.grad + at, g.ldg, 0, (int)g.np, at != 0);
                flush(g.grad + at + g.np, g.ldg, RUN, (int)g.np, at != 0);
            }
        }
    }
}

template <int HALF, int TN, int TM, int WN, int WM, int OUT>
__global__ __launch_bounds__(WN * WM * 64) void k_gemm(const Gemm g) {
    product<HALF, TN, TM, WN, WM, OUT>(g);
}

template <int HALF, int TN, int TM, int WN, int WM, int OUT>
int launch(const Gemm& g, hipStream_t st) {
    constexpr int TNE = OUT == OUT_GATED || OUT == OUT_GRAD ? TN / 2 : TN;
    const int64_t nt = (g.n + TNE - 1) / TNE, mt = (g.m + TM - 1) / TM;
    const int64_t groups = nt * mt * (OUT == OUT_PART ? g.pieces * (g.w1 ? 2 : 1) : 1);
    if (groups > INT32_MAX) return fail(SPA_ERR_ARG, "product: %d x %d outputs are too many", g.m, g.n);
    hipLaunchKernelGGL((k_gemm<HALF, TN, TM, WN, WM, OUT>), dim3((unsigned)groups), dim3(WN * WM * 64), 0, st, g);
    SPA_HIP_TRY(hipGetLastError());
    return SPA_OK;
}

// The pieces of k joined in their order, and what the one-launch forms do with the sums. Four columns a lane, AT
// pieces' loads under way at once.
template <int OUT>
__global__ __launch_bounds__(256) void k_join(const Gemm g) {
    constexpr bool TWO = OUT == OUT_GATED || OUT == OUT_GRAD;
    constexpr int AT = 4;
    const int width = OUT == OUT_GRAD ? (int)g.np : g.n, per = (width + 3) / 4;
    const int64_t total = (int64_t)g.m * per, size = (int64_t)g.m * g.n;
    for (int64_t at = blockIdx.x * 256ll + threadIdx.x; at < total; at += gridDim.x * 256ll) {
        const int m = (int)(at / per), n = (int)(at - (int64_t)m * per) * 4;
        float v[1 + TWO][4];
#pragma unroll
        for (int s = 0; s <= TWO; ++s) {
            const float* p = g.part + s * g.pieces * size + (int64_t)m * g.n + n;
#pragma unroll
            for (int c = 0; c < 4; ++c) v[s][c] = 0.f;
            for (int i = 0; i < g.pieces; i += AT) {
                f4 a[AT];
#pragma unroll
                for (int j = 0; j < AT; ++j) {                    // those beyond the last are dropped
                    const float* q = p + tmin(i + j, g.pieces - 1) * size;
                    if (n + 4 <= g.n) {
                        __builtin_memcpy(&a[j], q, 16);           // at any number's address
                    } else {
#pragma unroll
                        for (int c = 0; c < 4; ++c) a[j][c] = n + c < g.n ? q[c] : 0.f;
                    }
                }
#pragma unroll
                for (int j = 0; j < AT; ++j)
                    if (i + j < g.pieces)
#pragma unroll
                        for (int c = 0; c < 4; ++c) v[s][c] += a[j][c];
            }
        }
        if constexpr (OUT != OUT_GRAD) {
            uint16_t h[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                float a = v[0][c];
                if constexpr (TWO) a = act_value(a, g.act) * v[1][c];
                h[c] = narrow(a, g.kind);
            }
            uint16_t* y = g.y + (int64_t)m * g.ldy + n;
            if (n + 4 <= g.n) {
                __builtin_memcpy(y, h, 8);
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (n + c < g.n) y[c] = h[c];
            }
        } else {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int ni = n + c;
                float value = 0.f, slope = 0.f, d = 0.f;
                if (ni < g.n) {
                    act_both(v[0][c], g.act, value, slope);
                    d = wide(g.dh[(int64_t)m * g.ldh + ni], g.kind);
                }
                const int ge = g.ge ? g.ge[m] : 0;
                const int e0 = g.we0 && ni < g.n ? g.we0[ni] : 0, e1 = g.we1 && ni < g.n ? g.we1[ni] : 0;
                const float u = v[1][c];
                if (ni < width) {
                    uint16_t* y = g.grad + (int64_t)m * g.ldg + ni;
                    y[0] = narrow(ni < g.n ? ldexpf(d * u * slope, e0 - ge) : 0.f, g.half);
                    y[g.np] = narrow(ni < g.n ? ldexpf(d * value, e1 - ge) : 0.f, g.half);
                    if (g.twice) {
                        y[2 * g.np] = (uint16_t)finite2(y[0]);
                        y[3 * g.np] = (uint16_t)finite2(y[g.np]);
                    }
                }
            }
        }
    }
}

// What a product takes: the larger the tile, the less time for its work, but the device has 256 compute units and
// waits for its last round. A round's time in units of 1/100 us on one MI355X, for each 64 k and for its beginning
// and end: 256 x 256 162 and 1000; 128 x 128, two to a unit, 113 and 900, alone on it 83 and 600 (256 x 128 took 111,
// no more for its work than 128 x 128). In pieces of k, where there are too few tiles: their sums leave as float32
// (1500 or 700 a round), each adds 8 bytes of traffic an output and matrix (about 5 TB/s), and there is the joining
// launch.
enum Tile { SMALL, LARGE };
struct Plan {
    int tile;
    int pieces;
    int64_t cost;
};
int64_t tile_time(int tile, int64_t n, int64_t m, int64_t times, int64_t steps, bool part) {
    const int64_t t = tile == SMALL ? 128 : 256, tiles = (n + t - 1) / t * ((m + t - 1) / t) * times;
    const int64_t out = part ? (tile == LARGE ? 1500 : 700) : 0;
    if (tile == LARGE) return (tiles + 255) / 256 * (steps * 162 + 1000 + out);
    return tiles <= 256 ? steps * 83 + 600 + out : (tiles + 511) / 512 * (steps * 113 + 900 + out);
}
Plan plan(const Gemm& g) {
    const int64_t steps = g.k / BK, m = g.m, n = g.n, matrices = g.w1 ? 2 : 1;
    Plan best{LARGE, 1, INT64_MAX};
    for (int tile = LARGE; tile >= SMALL; --tile) {
        const int64_t whole = tile_time(tile, n * matrices, m, 1, steps, false);
        if (whole < best.cost) best = Plan{tile, 1, whole};
        for (int p = 2; p <= g.most && p * 4 <= steps; ++p) {
            // in pieces the two matrices are products of their own
            const int64_t c = tile_time(tile, n, m, matrices * p, (steps + p - 1) / p, true) + 600 + m * n * matrices * 8 * p / 50000;
            if (c < best.cost) best = Plan{tile, p, c};
        }
    }
    return best;
}

template <int HALF, int OUT>
int launch_tile(int tile, const Gemm& g, hipStream_t st) {
    return tile == LARGE ? launch<HALF, 256, 256, 2, 4, OUT>(g, st) : launch<HALF, 128, 128, 2, 2, OUT>(g, st);
}

template <int HALF, int OUT>
int pick(const Gemm& g, hipStream_t st) {
    const Plan p = plan(g);
    if (p.pieces > 1) {
        Gemm q = g;
        q.pieces = p.pieces;
        const int rc = launch_tile<HALF, OUT_PART>(p.tile, q, st);
        if (rc) return rc;
        const int64_t groups = ((int64_t)g.m * ((OUT == OUT_GRAD ? g.np : g.n) + 3) / 4 + 255) / 256;
        hipLaunchKernelGGL((k_join<OUT>), dim3((unsigned)(groups < 16384 ? groups : 16384)), dim3(256), 0, st, q);
        SPA_HIP_TRY(hipGetLastError());
        return SPA_OK;
    }
    return launch_tile<HALF, OUT>(p.tile, g, st);
}

template <int HALF>
int form(const Gemm& g, hipStream_t st) {
    if (g.grad) return pick<HALF, OUT_GRAD>(g, st);
    if (g.w1) return pick<HALF, OUT_GATED>(g, st);
    return g.ex.low ? pick<HALF, OUT_LOW>(g, st) : pick<HALF, OUT_PLAIN>(g, st);
}

}  // namespace

int64_t gemm_part(const Gemm& g) {
    Gemm q = g;
    q.most = GEMM_PIECES;
    const Plan p = plan(q);
    return p.pieces > 1 ? (int64_t)p.pieces * (g.w1 ? 2 : 1) * g.m * g.n : 0;
}

int64_t gemm_cost(const Gemm& g) {
    Gemm q = g;
    q.most = GEMM_PIECES;
    return plan(q).cost;
}

int gemm_pieces(const Gemm& g, hipStream_t st) {
    return g.half == SRC_BF16 ? launch<SRC_BF16, 128, 128, 2, 2, OUT_PART>(g, st) : launch<SRC_F16, 128, 128, 2, 2, OUT_PART>(g, st);
}

int gemm(const Gemm& g, hipStream_t st) { return g.half == SRC_BF16 ? form<SRC_BF16>(g, st) : form<SRC_F16>(g, st); }

}  // namespace lin
}  // namespace spa
