// Products of many 4-bit rows with 4-bit weights, whole or by expert.
//
// A workgroup computes TN weight rows x TM input rows, both by steps of 256 of k: 128 bytes of a row's codes. Codes go from
// HBM / L2 straight to LDS, into one of two buffers while the other is multiplied; LDS rows are 128 bytes too, their
// eight 16-byte blocks stored at block ^ (row / 2 & 7), so that a fragment read's 16 rows lie in 16 different places of the
// 256 bytes that LDS serves at once. Half h of a wave's lanes takes block 4 h + u of a step in instruction u: the four
// scales of its blocks are then one word, read once a step, whose bytes the instruction picks. Scales come four steps at a
// time, a quarter of the next four in each step: 32 bytes of a row, where 8 would fetch a whole line each step.
// Weights are the instruction's first operand: a lane then holds four consecutive outputs of a row. For the gated form half
// of the TN rows are the gate's and half the same rows of the up projection.
#include "../../include/seedpack_amd.h"
#include "launch.h"
#include "mx4.h"
#include "mx4_tiles.h"

#include <type_traits>

namespace spa {
namespace mx {
namespace {

using lin::f4;
using lin::f16v;
using lin::u4;
typedef int v8i __attribute__((ext_vector_type(8)));
typedef __amdgpu_buffer_rsrc_t rsrc;
typedef __attribute__((address_space(3))) void* lptr;

template <int U> __device__ __forceinline__ f16v mul(u4 w, u4 x, f16v c, uint32_t ws, uint32_t xs) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(v8i{(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0},
                                                           v8i{(int)x[0], (int)x[1], (int)x[2], (int)x[3], 0, 0, 0, 0}, c, 4, 4, U, (int)ws, U, (int)xs);
}

enum Out { OUT_PLAIN, OUT_GATED, OUT_PART };                  // PART: float32 sums of a piece of k of one matrix

// An activation's value by the hardware's 2^x and 1 / x, both good to an ulp. Outputs of 16 bits do without the logit's second
// part: its rounding in units of log2 costs |logit| 2^-24 of the result, a 64th of their half step at most, and with two parts the
// outputs of 128 x 256 take 5 us, not 3. Outputs in float32 would show it (a gate of -80 was off by 60 2^-24).
template <int KIND, int ACT> __device__ __forceinline__ float act_of(float g) {
    if constexpr (KIND == SRC_F32) return lin::act_value(g, ACT);
    return g * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504f * lin::act_logit(g, ACT)));
}

template <int TN, int TM, int WN, int WM, int OUT>
__device__ __forceinline__ void product(const Product& p) {
    constexpr bool TWO = OUT == OUT_GATED;
    constexpr int NW = WN * WM;                              // waves
    constexpr int TNE = TWO ? TN / 2 : TN;                   // output columns of the tile
    constexpr int FN = TN / WN / 32, FM = TM / WM / 32;      // 32 x 32 fragments of a wave
    constexpr int ROWS = TN + TM;
    constexpr int LOADS = ROWS / 8 / NW;                     // 8 rows by one load of a wave
    static_assert(TNE % (8 * NW) == 0 && 32 * NW == TN && TM == TN && TNE % 32 == 0 && (!TWO || FN % 2 == 0), "tile shape");
    constexpr int COLS = TNE / WN;                           // a wave's columns on their way out
    constexpr int STAGES = 2 * ROWS * 128, SCALES = 2 * ROWS * 32, OUTS = NW * 32 * (COLS + 4) * 4;
    __shared__ __align__(16) uint8_t mem[STAGES + SCALES > OUTS ? STAGES + SCALES : OUTS];
    uint8_t* const smem = mem + STAGES;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // Tiles are dealt so that each of the 8 XCDs, which take workgroups in turn, has a run of neighbours: its L2 then
    // serves their shared rows. By expert a tile of inputs is followed through all of its expert's weights.
    const Tiles tiles = tiles_of(p, TM);
    const int nt = (p.n + TNE - 1) / TNE, mt = tmin(tiles.total, most_tiles(p, TM));   // more only where starts do not rise
    const int total = nt * mt;
    int id, piece = 0;
    bool second = false;                                     // of the gated form's two matrices, each a product of its own
    {
        const int all = OUT == OUT_PART ? total * p.pieces * (p.w1c ? 2 : 1) : total;
        const int q = all / 8, r = all % 8, xcd = blockIdx.x & 7, at = blockIdx.x >> 3;
        if (at >= q + (xcd < r)) return;
        id = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + at;
    }
    int from = 0, steps = p.pitch / 8;                       // in steps of 256 of k
    if (OUT == OUT_PART) {
        piece = id / total;
        id -= piece * total;
        second = piece >= p.pieces;
        const int i = second ? piece - p.pieces : piece;
        from = steps * i / p.pieces;
        steps = steps * (i + 1) / p.pieces - from;
    }
    int n0;
    Tile t;
    if (p.experts) {
        t = tile_at(p, tiles, id / nt, TM);
        n0 = id % nt * TNE;
    } else {
        constexpr int GROUP = 8;
        const int band = id / (GROUP * nt), in = id - band * GROUP * nt, height = tmin(GROUP, mt - band * GROUP);
        t = tile_at(p, tiles, band * GROUP + in % height, TM);
        n0 = in / height * TNE;
    }

    const uint32_t row16 = (uint32_t)p.pitch * 16;
    const int64_t wfirst = (int64_t)t.expert * p.n + n0, xfirst = p.experts ? 0 : t.first;
    // What the lane's input rows are, and its output's: each asked for at its own use, they would wait for memory one by one, so
    // all are asked for here, and waited for behind the first fetches of weights.
    constexpr int LW = TN / 8 / NW, LX = LOADS - LW;         // loads of weights, of inputs
    const int wn = wave % WN, wm = wave / WN;
    static_assert(TM / WM == 64, "tile shape");
    int row[LX + 2];                                         // those of its loads, of its scales, and the output's
    {
        const int lr = lane >> 3;
#pragma unroll
        for (int j = 0; j < LX + 2; ++j) {
            const int r = j < LX ? (j * NW + wave) * 8 + lr : j == LX ? wave * 32 + (lane >> 1) : wm * 64 + lane;
            row[j] = tmin(r, t.rows - 1);                    // rows behind the last are the last
        }
        if (p.experts) {
#pragma unroll
            for (int j = 0; j < LX + 2; ++j) row[j] = p.order[t.first + row[j]];
        }
    }
    // a weights' row of the tile, from the first
    auto weight_row = [&](int r) { return (uint32_t)tmin(r - (TWO && r >= TNE ? TNE : 0), p.n - 1 - n0); };
    uint32_t off[LOADS], soff[2];
    const int lr = lane >> 3, chunk = (lane & 7) ^ ((lr >> 1) + 4 * (wave & 1));
#pragma unroll
    for (int j = 0; j < LW; ++j) off[j] = weight_row((j * NW + wave) * 8 + lr) * row16 + 16 * chunk;
    // A wave's scales: 32 of the weights' rows by one load, 32 of the inputs' by another, two pieces of 16 bytes a row; the
    // pieces of every other run of 8 rows lie exchanged, for a fragment's reads.
    soff[0] = weight_row(wave * 32 + (lane >> 1)) * (uint32_t)p.pitch;
    const int spiece = 16 * ((lane & 1) ^ (lane >> 4 & 1));
    constexpr int RAW = 0x00027000;                               // a plain buffer of bytes
    auto buffer = [&](const uint8_t* b, int64_t first, int64_t row) { return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(b + first * row), 0, -1, RAW); };
    const uint8_t *const wc = second ? p.w1c : p.w0c, *const ws = second ? p.w1s : p.w0s;
    const rsrc rw0 = buffer(wc + from * 128, wfirst, row16), rw1 = TWO ? buffer(p.w1c, wfirst, row16) : rw0, rx = buffer(p.xc + from * 128, xfirst, row16);
    const rsrc sw = buffer((TWO && wave * 32 >= TNE ? p.w1s : ws) + from * 8, wfirst, p.pitch), sx = buffer(p.xs + from * 8, xfirst, p.pitch);
    const int left = p.pitch - 8 * from;                     // scales of a row from here on
    auto fetch = [&](int buf, int kt, int j0, int j1) {
#pragma unroll
        for (int j = j0; j < j1; ++j) {
            const rsrc r = j * NW * 8 >= TN ? rx : (TWO && j * NW * 8 >= TNE ? rw1 : rw0);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lptr)(mem + buf * ROWS * 128 + (j * NW + wave) * 8 * 128), 16, off[j], kt * 128, 0, 0);
        }
    };
    // half of the scales of steps 4 g .. 4 g + 3, the weights' or the inputs'. A piece that would end 8 bytes behind its row
    // is taken 8 bytes early (odd_end); those behind the row's last are others. A row that has only 8: word by word.
    auto fetch_scales = [&](int g, auto half) {
        constexpr int H = decltype(half)::value;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(H ? sx : sw, (lptr)(smem + (g & 1) * ROWS * 32 + (H * TN + wave * 32) * 32), 16,
                                                 soff[H] + (uint32_t)tmin(32 * g + spiece, left - 16), 0, 0, 0);
    };
    auto fetch_words = [&](auto half) {
        constexpr int H = decltype(half)::value;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t row = (uint32_t)__shfl((int)soff[H], 16 * i + 2 * (lane >> 3));
            const int piece = (lane >> 2 & 1) ^ (i & 1);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(H ? sx : sw, (lptr)(smem + (H * TN + wave * 32 + 8 * i) * 32), 4,
                                                     row + (uint32_t)tmin(16 * piece + 4 * (lane & 3), left - 4), 0, 0, 0);
        }
    };
    const std::integral_constant<int, 0> H0;
    const std::integral_constant<int, 1> H1;
    auto odd_end = [&](int kt) { return 16 * (kt >> 1) > left - 16 && left > 8 ? 8 : 0; };

    const int fr = lane & 31, fk = lane >> 5;                // a fragment's row and its half of 64 k
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

    u4 fa[2][FN], fb[2][FM];
    uint32_t sa[FN], sb[FM], na[FN], nb[FM];
    auto read = [&](int buf, int part, int to) {
        const uint8_t* const b = mem + buf * ROWS * 128;
#pragma unroll
        for (int i = 0; i < FN; ++i) fa[to][i] = *reinterpret_cast<const u4*>(b + arow[i] * 128 + ((4 * fk + part) ^ ((arow[i] >> 1) & 7)) * 16);
#pragma unroll
        for (int i = 0; i < FM; ++i) fb[to][i] = *reinterpret_cast<const u4*>(b + brow[i] * 128 + ((4 * fk + part) ^ ((brow[i] >> 1) & 7)) * 16);
    };
    auto read_scales = [&](int kt) {
        const uint8_t* const b = smem + (kt >> 2 & 1) * ROWS * 32 + (kt & 1) * 8 + odd_end(kt) + 4 * fk;
        auto at = [&](int row) { return *reinterpret_cast<const uint32_t*>(b + row * 32 + ((kt >> 1 & 1) ^ (row >> 3 & 1)) * 16); };
#pragma unroll
        for (int i = 0; i < FN; ++i) na[i] = at(arow[i]);
#pragma unroll
        for (int i = 0; i < FM; ++i) nb[i] = at(brow[i]);
    };
    // One step; N1, N2: there is a next one, and one after that. Fragments are read one part ahead of their use; in a step's
    // last part the other buffer's first are read. Before it every wave's fetches into that buffer have arrived and
    // every wave has read the last of this one: one barrier a step orders both. A wave none of whose rows the tile has (ACTIVE
    // false) fetches and meets the others.
    constexpr int EARLY = LOADS / 2;
    auto tile_step = [&](int kt, auto n1, auto n2, auto act) {
        constexpr bool N1 = decltype(n1)::value, N2 = decltype(n2)::value, ACTIVE = decltype(act)::value;
        const int buf = kt & 1;
        if (ACTIVE) {
#pragma unroll
            for (int i = 0; i < FN; ++i) sa[i] = na[i];
#pragma unroll
            for (int i = 0; i < FM; ++i) sb[i] = nb[i];
        }
        auto part = [&](auto u) {
            constexpr int U = decltype(u)::value;
            constexpr bool last = U == 3;
            auto products = [&](int i0, int i1) {
#pragma unroll
                for (int i = i0; i < i1; ++i)
#pragma unroll
                    for (int j = 0; j < FM; ++j) acc[i][j] = mul<U>(fa[U & 1][i], fb[U & 1][j], acc[i][j], sa[i], sb[j]);
            };
            constexpr int AHEAD = FN / 4 > 0 ? FN / 4 : 1;
            if (last && N1) {
                // some of the part's products are under way while the waves meet
                if (ACTIVE) products(0, AHEAD);
                __builtin_amdgcn_sched_barrier(0);
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            }
            if (ACTIVE) {
                if (!last) read(buf, U + 1, (U + 1) & 1);
                else if (N1) {
                    read(buf ^ 1, 0, 0);
                    read_scales(kt + 1);
                }
            }
            if (U == 0 && N1) fetch(buf ^ 1, kt + 1, EARLY, LOADS);
            if (last && N2) {
                fetch(buf, kt + 2, 0, EARLY);
                if (((kt + 1) & 3) == 0) fetch_scales((kt + 1) / 4 + 1, H0);
                if (((kt + 1) & 3) == 1) fetch_scales((kt + 1) / 4 + 1, H1);
            }
            if (ACTIVE) {
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
        part(std::integral_constant<int, 0>());
        part(std::integral_constant<int, 1>());
        part(std::integral_constant<int, 2>());
        part(std::integral_constant<int, 3>());
    };
    auto sums = [&](auto act) {
        if (decltype(act)::value) {
            read(0, 0, 0);
            read_scales(0);
        }
        for (int kt = 0; kt < steps - 2; ++kt) tile_step(kt, std::true_type(), std::true_type(), act);
        if (steps > 1) tile_step(steps - 2, std::true_type(), std::false_type(), act);
        tile_step(steps - 1, std::false_type(), std::false_type(), act);
    };
    fetch(0, 0, 0, LW);
    if (left > 8) fetch_scales(0, H0);
    else fetch_words(H0);
    int out_rows = row[LX + 1] + t.first;                     // of the wave, one a lane
    if (p.experts) {
        out_rows = (uint32_t)row[LX + 1] < (uint32_t)p.m ? row[LX + 1] : -1;
        input_rows<LX + 1>(p, row);
    }
#pragma unroll
    for (int j = 0; j < LX; ++j) off[LW + j] = (uint32_t)row[j] * row16 + 16 * chunk;
    soff[1] = (uint32_t)row[LX] * (uint32_t)p.pitch;
    if (left > 8) fetch_scales(0, H1);
    else fetch_words(H1);
    fetch(0, 0, LW, LOADS);
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    if (steps > 1) {
        fetch(1, 1, 0, EARLY);
        fetch_scales(1, H0);
    }
    const bool active = wm * (TM / WM) < t.rows;
    if (active) sums(std::true_type());
    else sums(std::false_type());

    // Lane: input row (lane & 31) of a fragment; register 4 q + c: weight row 8 q + 4 (lane >> 5) + c. By way of LDS, which
    // the loop is done with, 32 input rows at a time leave in runs of the wave's columns.
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (!active) return;
    constexpr int PITCH = COLS + 4;
    float* const stage = reinterpret_cast<float*>(mem) + wave * 32 * PITCH;
    // (a body for each activation and type: with both activations worked out for every output, or choices among types, the
    // outputs of 256 x 128 gated take 6 us)
    auto leave = [&](auto kind, auto act) {
        constexpr int KIND = decltype(kind)::value, ACT = decltype(act)::value;
        const bool wide16 = (p.ldy * (KIND == SRC_F32 ? 4 : 2) & 15) == 0 && (reinterpret_cast<uintptr_t>(p.y) & 15) == 0;
#pragma unroll
        for (int j = 0; j < FM; ++j) {
#pragma unroll
            for (int i = 0; i < (TWO ? FN / 2 : FN); ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    f4 v;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        v[c] = acc[i][j][4 * q + c];
                        if (TWO) v[c] = act_of<KIND, ACT>(v[c]) * acc[i + (TWO ? FN / 2 : 0)][j][4 * q + c];
                    }
                    *reinterpret_cast<f4*>(stage + fr * PITCH + 32 * i + 8 * q + 4 * fk) = v;
                }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            const int m0 = wm * (TM / WM) + 32 * j;
            for (int u = lane; u < 32 * (COLS / 8); u += 64) {
                const int r = u / (COLS / 8), c = u % (COLS / 8) * 8, n = n0 + wn * COLS + c;
                const int64_t row = OUT == OUT_PART ? 0 : __shfl(out_rows, 32 * j + r);
                if (m0 + r >= t.rows || n >= p.n || row < 0) continue;
                const f4 a = *reinterpret_cast<const f4*>(stage + r * PITCH + c), b = *reinterpret_cast<const f4*>(stage + r * PITCH + c + 4);
                const bool whole = n + 8 <= p.n;
                if constexpr (KIND == SRC_F32) {
                    float* const y = OUT == OUT_PART ? p.part + ((int64_t)piece * p.m + t.first + m0 + r) * p.n + n : static_cast<float*>(p.y) + row * p.ldy + n;
                    if (whole && wide16 && OUT != OUT_PART) {
                        __builtin_nontemporal_store(a, reinterpret_cast<f4*>(y));
                        __builtin_nontemporal_store(b, reinterpret_cast<f4*>(y) + 1);
                    } else if (whole) {
                        __builtin_memcpy(y, &a, 16);              // at any number's address
                        __builtin_memcpy(y + 4, &b, 16);
                    } else {
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            if (n + k < p.n) y[k] = k < 4 ? a[k & 3] : b[k & 3];
                    }
                } else {
                    uint16_t* const y = static_cast<uint16_t*>(p.y) + row * p.ldy + n;
                    const u4 v = {lin::narrow2(a[0], a[1], KIND), lin::narrow2(a[2], a[3], KIND), lin::narrow2(b[0], b[1], KIND), lin::narrow2(b[2], b[3], KIND)};
                    if (whole && wide16) {
                        __builtin_nontemporal_store(v, reinterpret_cast<u4*>(y));
                    } else if (whole) {
                        __builtin_memcpy(y, &v, 16);
                    } else {
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            if (n + k < p.n) y[k] = (uint16_t)(v[k >> 1] >> (16 * (k & 1)));
                    }
                }
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
    };
    auto of_kind = [&](auto kind) {
        if (TWO && p.act == lin::ACT_GELU) leave(kind, std::integral_constant<int, lin::ACT_GELU>());
        else leave(kind, std::integral_constant<int, lin::ACT_SILU>());
    };
    if (OUT == OUT_PART || p.kind == SRC_F32) of_kind(std::integral_constant<int, SRC_F32>());
    else if (p.kind == SRC_BF16) of_kind(std::integral_constant<int, SRC_BF16>());
    else of_kind(std::integral_constant<int, SRC_F16>());
}

template <int TN, int TM, int WN, int WM, int OUT>
__global__ __launch_bounds__(WN * WM * 64) void k_product(const Product p) {
    product<TN, TM, WN, WM, OUT>(p);
}

// The pieces' sums added in their order, four columns a lane; by expert row i is the slot that the order names
template <bool TWO>
__global__ __launch_bounds__(256) void k_join_pieces(const Product p) {
    const int per = (p.n + 3) / 4;
    const int64_t id = blockIdx.x * 256ll + threadIdx.x;
    const int64_t i = id / per;
    const int n = (int)(id - i * per) * 4;
    if (i >= (p.experts ? tmin(p.starts[p.experts], p.m) : p.m)) return;
    const int64_t row = output_row(p, (int)i);
    if (row < 0) return;
    const int64_t size = (int64_t)p.m * p.n;
    const bool whole = n + 4 <= p.n;
    f4 v[1 + TWO];
#pragma unroll
    for (int s = 0; s <= TWO; ++s) {
        v[s] = f4{0, 0, 0, 0};
        for (int k = 0; k < p.pieces; ++k) {
            const float* const q = p.part + (s * p.pieces + k) * size + i * p.n + n;
            f4 a = {0, 0, 0, 0};
            if (whole) {
                __builtin_memcpy(&a, q, 16);                      // at any number's address
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (n + c < p.n) a[c] = q[c];
            }
            v[s] += a;
        }
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        if (n + c >= p.n) continue;
        const float f = TWO ? lin::act_value(v[0][c], p.act) * v[TWO][c] : v[0][c];
        if (p.kind == SRC_F32) static_cast<float*>(p.y)[row * p.ldy + n + c] = f;
        else static_cast<uint16_t*>(p.y)[row * p.ldy + n + c] = lin::narrow(f, p.kind);
    }
}

template <int TN, int TM, int WN, int WM, int OUT> int launch(const Product& p, hipStream_t st) {
    constexpr int TNE = OUT == OUT_GATED ? TN / 2 : TN;
    const int64_t groups = (int64_t)((p.n + TNE - 1) / TNE) * most_tiles(p, TM) * (OUT == OUT_PART ? p.pieces * (p.w1c ? 2 : 1) : 1);
    if (!one_launch(groups, WN * WM * 64)) return fail(SPA_ERR_ARG, "product: %d x %d outputs are too many", p.m, p.n);
    hipLaunchKernelGGL((k_product<TN, TM, WN, WM, OUT>), dim3((unsigned)groups), dim3(WN * WM * 64), 0, st, p);
    SPA_HIP_TRY(hipGetLastError());
    return SPA_OK;
}

}  // namespace

int product_many(const Product& p, bool large, hipStream_t st) {
    if (p.pieces > 1) {
        const int64_t workgroups = ((int64_t)p.m * ((p.n + 3) / 4) + 255) / 256;
        if (!one_launch(workgroups, 256)) return fail(SPA_ERR_ARG, "product: %d x %d outputs are too many", p.m, p.n);
        const int rc = launch<128, 128, 2, 2, OUT_PART>(p, st);
        if (rc) return rc;
        const dim3 grid((unsigned)workgroups);
        if (p.w1c) hipLaunchKernelGGL(k_join_pieces<true>, grid, dim3(256), 0, st, p);
        else hipLaunchKernelGGL(k_join_pieces<false>, grid, dim3(256), 0, st, p);
        SPA_HIP_TRY(hipGetLastError());
        return SPA_OK;
    }
    if (large) return p.w1c ? launch<256, 256, 2, 4, OUT_GATED>(p, st) : launch<256, 256, 2, 4, OUT_PLAIN>(p, st);
    return p.w1c ? launch<128, 128, 2, 2, OUT_GATED>(p, st) : launch<128, 128, 2, 2, OUT_PLAIN>(p, st);
}

}  // namespace mx
}  // namespace spa
