// The products with packed weights behind the C ABI: arguments checked, the form chosen by sizes and types,
// the workspace laid out. Nothing is allocated and nothing waits; every launch goes to the caller's stream.
#include "../../include/seedpack_amd.h"
#include "launch.h"
#include "linear.h"

namespace spa {
namespace lin {
namespace {

// Rows of the inner matrices lie 128 bytes more than whole steps apart: at powers of two, the rows of a tile share few
// of the memory's channels (4096 x 4096 x 24576: 660 to 616 us)
constexpr int64_t PAD = 64;
int64_t up64(int64_t v) { return (v + 63) / 64 * 64; }

// a workspace handed out in pieces of whole 256 bytes; with no memory behind it, only counted
struct Work {
    uint8_t* base;
    uint64_t used = 0;
    template <typename T> T* take(int64_t n) {
        T* p = reinterpret_cast<T*>(base + used);
        used += ((uint64_t)n * sizeof(T) + 255) / 256 * 256;
        return p;
    }
};

bool is16(int type) { return type == 1 || type == 30; }
int kind_of(int type) { return type == 1 ? SRC_F16 : SRC_BF16; }

// A tile's rows are fetched at 32-bit offsets from its first: 255 rows of four inner matrices' or twice the columns
// and their last byte have to stay below 2^32.
constexpr int64_t MOST_COLS = 4000000, MOST_INNER = 2000000;

int check_weight(const char* who, int type, int64_t n, int64_t k) {
    if (!is16(type) && !type_qk(type)) return fail(SPA_ERR_TYPE, "%s: weights of type %d are not supported", who, type);
    if (n < 0 || k <= 0 || n > INT32_MAX - 256 || k > MOST_COLS)
        return fail(SPA_ERR_ARG, "%s: bad weight shape %lld x %lld", who, (long long)n, (long long)k);
    if (!is16(type) && k % type_qk(type))
        return fail(SPA_ERR_ARG, "%s: row of %lld not a multiple of %d (type %d)", who, (long long)k, type_qk(type), type);
    return SPA_OK;
}
int check_rows(const char* who, int kind, int64_t m, int64_t k, int64_t stride) {
    if (kind != SPA_SRC_BF16 && kind != SPA_SRC_F16) return fail(SPA_ERR_TYPE, "%s: inputs of kind %d (BF16 and F16 are taken)", who, kind);
    if (m < 0 || m > INT32_MAX - 256 || stride < k) return fail(SPA_ERR_ARG, "%s: bad shape %lld x %lld, stride %lld", who, (long long)m, (long long)k, (long long)stride);
    return SPA_OK;
}
bool on(const void* p, uintptr_t unit) { return (reinterpret_cast<uintptr_t>(p) & (unit - 1)) == 0; }
int check_weight_at(const char* who, int type, const void* w) {
    // 16-bit weights are fetched sixteen bytes at a time; blocks lie at any byte
    if (is16(type) && !on(w, 16)) return fail(SPA_ERR_ARG, "%s: 16-bit weights not 16-byte aligned", who);
    return SPA_OK;
}
int check_work(const char* who, const void* work, uint64_t have, uint64_t need) {
    if (need && (!work || !on(work, 256) || have < need))
        return fail(SPA_ERR_ARG, "%s: needs a 256-byte aligned workspace of %llu bytes, got %llu", who, (unsigned long long)need, (unsigned long long)(work ? have : 0));
    return SPA_OK;
}
int64_t weight_bytes(int type, int64_t n, int64_t k) { return is16(type) ? 2 * n * k : n * (k / type_qk(type)) * type_bs(type); }

// the operands of a product as its kernels take them
struct Operands {
    const uint16_t *x = nullptr, *w0 = nullptr, *w1 = nullptr;
    int64_t ldx = 0, ldw = 0;
    int half = 0;
    int64_t kp = 0, rest = 0;   // columns of the rows, and where the weights' second parts begin (0: none)
    int32_t *xe = nullptr, *we0 = nullptr, *we1 = nullptr;
    float *norm = nullptr, *n0 = nullptr, *n1 = nullptr;
};

// Inputs and weights brought into the form of the many-rows product. Where both are of one 16-bit type they
// are used as they lie, or copied where rows are not whole 128-byte steps at 16-byte addresses; otherwise
// both become binary16 rows, beside F16 inputs the weights of block types in two parts. `run` false only lays out
// the workspace (for the widest case).
int operands(Work& wk, bool run, int type, const void* w0, const void* w1, int64_t n, int64_t k, int kind, const void* x, int64_t m,
             int64_t ldx, bool bounds, Operands& o, hipStream_t st) {
    const int64_t kp = up64(k);
    const bool same = is16(type) && kind_of(type) == kind;
    o.half = same ? kind : SRC_F16;
    const bool both = !same && !is16(type) && kind == SRC_F16;
    const int64_t ldd = same ? kp : (both ? 2 : 1) * kp + PAD;
    o.kp = both ? 2 * kp : kp;
    o.rest = both ? kp : 0;
    uint16_t* xp = wk.take<uint16_t>(m * ldd);
    int rc;
    if (same) {
        o.x = (const uint16_t*)x;
        o.ldx = ldx;
        if (run && (kp != k || !on(x, 16) || ldx % 8 || ldx > MOST_COLS)) {
            if ((rc = pack_rows((const uint16_t*)x, ldx, m, k, xp, kp, st))) return rc;
            o.x = xp;
            o.ldx = kp;
        }
        o.w0 = (const uint16_t*)w0;
        o.w1 = (const uint16_t*)w1;
        o.ldw = k;
        if (kp != k) {
            uint16_t* p0 = wk.take<uint16_t>(n * kp);
            uint16_t* p1 = w1 ? wk.take<uint16_t>(n * kp) : nullptr;
            if (run) {
                if ((rc = pack_rows(o.w0, k, n, k, p0, kp, st))) return rc;
                if (w1 && (rc = pack_rows(o.w1, k, n, k, p1, kp, st))) return rc;
            }
            o.w0 = p0;
            o.w1 = p1;
            o.ldw = kp;
        }
        return SPA_OK;
    }
    o.xe = wk.take<int32_t>(m);
    if (bounds) {
        o.norm = wk.take<float>(m);
        o.n0 = wk.take<float>(n);
        o.n1 = wk.take<float>(n);
    }
    if (run && (rc = half_rows((const uint16_t*)x, kind, ldx, m, k, xp, kp, ldd, o.xe, o.norm, both, st))) return rc;
    o.x = xp;
    o.ldx = o.ldw = ldd;
    for (int i = 0; i < (w1 ? 2 : 1); ++i) {
        uint16_t* p = wk.take<uint16_t>(n * ldd);
        int32_t* e = wk.take<int32_t>(n);
        const void* w = i ? w1 : w0;
        if (run) {
            rc = is16(type) ? half_rows((const uint16_t*)w, kind_of(type), k, n, k, p, kp, ldd, e, i ? o.n1 : o.n0, false, st)
                            : half_blocks(type, (const uint8_t*)w, n, k, p, kp, ldd, e, i ? o.n1 : o.n0, both, st);
            if (rc) return rc;
        }
        (i ? o.w1 : o.w0) = p;
        (i ? o.we1 : o.we0) = e;
    }
    return SPA_OK;
}

// Few rows: the weights as they lie. The inputs are copied where their rows are not whole steps of 32 at 16-byte
// addresses.
int few_operands(Work& wk, bool run, int type, const void* w0, const void* w1, int64_t n, int64_t k, const void* x, int64_t m,
                 int64_t ldx, Few& f, uint16_t*& frags, hipStream_t st) {
    const int64_t kp = (k + 31) / 32 * 32;
    frags = wk.take<uint16_t>(few_fragments(type, m, kp));
    uint16_t* xp = wk.take<uint16_t>(m * kp);
    int rc;
    f.x = (const uint16_t*)x;
    f.ldx = ldx;
    if (run && (kp != k || !on(x, 16) || ldx % 8)) {
        if ((rc = pack_rows(f.x, ldx, m, k, xp, kp, st))) return rc;
        f.x = xp;
        f.ldx = kp;
    }
    f.w0 = (const uint8_t*)w0;
    f.w1 = (const uint8_t*)w1;
    f.type = type;
    f.n = (int)n;
    f.k = (int)kp;
    f.m = (int)m;
    f.wbytes = weight_bytes(type, n, k);
    f.rowbytes = weight_bytes(type, 1, k);
    return SPA_OK;
}

Gemm gemm_of(const Operands& o, int64_t m, int64_t n) {
    Gemm g{};
    g.half = o.half;
    g.x = o.x;
    g.w0 = o.w0;
    g.w1 = o.w1;
    g.ldx = o.ldx;
    g.ldw = o.ldw;
    g.m = (int)m;
    g.n = (int)n;
    g.k = (int)o.kp;
    g.xe = o.xe;
    g.we0 = o.we0;
    g.we1 = o.we1;
    return g;
}

// the product with scratch for its pieces of k
int multiply(Gemm& g, Work& wk, bool run, hipStream_t st) {
    const int64_t part = gemm_part(g);
    g.part = wk.take<float>(part);
    g.most = part ? GEMM_PIECES : 1;
    return run ? gemm(g, st) : SPA_OK;
}

struct Project {
    int type;
    const void* w;
    int64_t n, k;
    int kind;
    const void* x;
    int64_t m, ldx;
    void* y;
    int64_t ldy;
    const void *a, *b;
    const float* scale;
    int64_t pool, rank;
    const int32_t* which;
};

// Many rows' first products as one product with every adapter of the pool, where it is small enough that
// the rows' other adapters cost less than reading x a few lanes at a time (2053 rows of 12288, 4 adapters of rank
// 64: 55 us row by row, 27 and 5 of picking): 128 x 128 tiles in pieces of k that fill the device, two to a compute unit. Tiles of
// adapters that none of their rows have are left out. Whole calls row by row and this way, BF16 with 1024 outputs, us:
//     k   rows    4 x 16     4 x 64    16 x 64    32 x 64 (width 2048)
//  1024    512    20  24     33  33     54  54     73  73
//  2048    128    24  28     31  30     51  49     74  73
//  2048    512    26  27     36  31     42  37     49  44
//  4096     65    28  29     40  30     57  47     83  73
//  4096   4096    61  62     81  71     82  83     96 106
// 12288     65    48  37     81  38     99  59    118  80
// 12288   4096   143 130    179 140    182 183    201 276
// (adapters of rank 16, whose rows form has one tile of them, gain nothing below 257 rows but from k = 12288)
int64_t low_as_product(const Project& p) {
    const int64_t width = p.pool * p.rank;
    if (p.m <= (p.k < 4096 || p.rank <= 16 ? 256 : FEW_ROWS) || width > 1024 || p.k % 64 || p.k < 2048) return 0;
    const int64_t tiles = (p.m + 127) / 128 * ((width + 127) / 128), pieces = tiles < 512 ? 512 / tiles : 1;
    return pieces < p.k / 256 ? pieces : p.k / 256;
}

// rows beyond whole tiles that the few-rows form takes, because the tiles they would need cost more: its weights at
// about 2 TB/s and two launches. The types whose few-rows form decodes in registers are left out.
int64_t tail_rows(const Gemm& g, int type) {
    if (!coded(type) && !is16(type)) return 0;
    const int64_t bytes = weight_bytes(type, g.n, g.k) * (g.w1 ? 2 : 1), extra = 1500 + bytes / 20000;
    int64_t best = 0, cost = gemm_cost(g);
    for (int tile = 256; tile >= 128; tile /= 2) {
        const int t = g.m % tile;
        if (t == 0 || t > 16 || t == g.m) continue;
        Gemm q = g;
        q.m = g.m - t;
        if (gemm_cost(q) + extra < cost) {
            best = t;
            cost = gemm_cost(q) + extra;
        }
    }
    return best;
}

int project(const Project& p, Work& wk, bool run, hipStream_t st) {
    Expand ex{};
    int rc;
    uint16_t* framed = nullptr;                                  // the fragments of a few-rows form, made beside low
    if (p.pool) {
        ex.rank = (int)p.rank;
        ex.rp = (int)((p.rank + 15) / 16 * 16);
        float* low = wk.take<float>(p.m * ex.rp);
        ex.low = low;
        ex.b = (const uint16_t*)p.b;
        ex.which = p.which;
        ex.pool = (int)p.pool;
        ex.kind = p.kind;
        ex.wide_b = p.rank % 8 == 0 && on(p.b, 16);
        const int64_t pieces = low_as_product(p);
        float* part = wk.take<float>(pieces * p.m * p.pool * p.rank);
        if (run && pieces && on(p.x, 16) && on(p.a, 16) && p.ldx % 8 == 0 && p.ldx <= MOST_COLS) {
            Gemm g{};
            g.half = p.kind;
            g.x = (const uint16_t*)p.x;
            g.ldx = p.ldx;
            g.w0 = (const uint16_t*)p.a;
            g.ldw = p.k;
            g.m = (int)p.m;
            g.n = (int)(p.pool * p.rank);
            g.k = (int)p.k;
            g.part = part;
            g.pieces = (int)pieces;
            g.which = p.which;
            g.rank = (int)p.rank;
            if ((rc = gemm_pieces(g, st))) return rc;
            if ((rc = low_pick(part, (int)pieces, p.scale, p.which, p.m, (int)p.pool, (int)p.rank, low, ex.rp, st))) return rc;
        } else {
            const int64_t frags = p.m <= FEW_ROWS && p.k % 32 == 0 ? few_fragments(p.type, p.m, p.k) : 0;
            uint16_t* to = wk.take<uint16_t>(frags);
            if (run && frags && on(p.x, 16) && p.ldx % 8 == 0) framed = to;
            if (run && (rc = low_rows((const uint16_t*)p.x, p.ldx, p.kind, p.m, p.k, (const uint16_t*)p.a, p.scale, p.which, (int)p.pool,
                                      (int)p.rank, low, ex.rp, Frags{framed, few_tiles(p.type, p.m), (int)p.k, p.type == 14}, st)))
                return rc;
        }
    }
    auto few_rows = [&](int64_t from, int64_t m) {
        Few f{};
        uint16_t* frags;
        const int r = few_operands(wk, run, p.type, p.w, nullptr, p.n, p.k, (const uint16_t*)p.x + from * p.ldx, m, p.ldx, f, frags, st);
        if (r || !run) return r;
        f.kind = p.kind;
        f.y = (uint16_t*)p.y + from * p.ldy;
        f.ldy = p.ldy;
        f.ex = ex;
        if (ex.low) {
            f.ex.low += from * ex.rp;
            f.ex.which += from;
        }
        f.framed = framed != nullptr;
        return few(f, framed ? framed : frags, st);
    };
    if (p.m <= few_limit(p.type)) {
        for (int64_t at = 0; at < p.m; at += FEW_ROWS)
            if ((rc = few_rows(at, p.m - at < FEW_ROWS ? p.m - at : FEW_ROWS))) return rc;
        return SPA_OK;
    }
    Operands o;
    if ((rc = operands(wk, run, p.type, p.w, nullptr, p.n, p.k, p.kind, p.x, p.m, p.ldx, false, o, st))) return rc;
    Gemm g = gemm_of(o, p.m, p.n);
    g.kind = p.kind;
    g.y = (uint16_t*)p.y;
    g.ldy = p.ldy;
    g.ex = ex;
    const int64_t tail = tail_rows(g, p.type);
    g.m -= (int)tail;
    if ((rc = multiply(g, wk, run, st))) return rc;
    return tail ? few_rows(p.m - tail, tail) : SPA_OK;
}

struct Gated {
    int type;
    const void *gate, *up;
    int64_t n, k;
    int kind;
    const void* x;
    int64_t m, ldx;
    int act;
    void* h;
    int64_t ldh;
    const void* dh;             // the backward form from here on: dh has rows of ldh too
    void *dx, *dgate, *dup;
    int64_t lddx;
};
// no pointer of a counted layout is read; the second matrix only has to be there
const void* const SOME = reinterpret_cast<const void*>(256);

int gated(const Gated& p, Work& wk, bool run, hipStream_t st) {
    int rc;
    const void* up = run ? p.up : SOME;
    auto few_rows = [&](int64_t from, int64_t m) {
        Few f{};
        uint16_t* frags;
        const int r = few_operands(wk, run, p.type, p.gate, up, p.n, p.k, (const uint16_t*)p.x + from * p.ldx, m, p.ldx, f, frags, st);
        if (r || !run) return r;
        f.kind = p.kind;
        f.y = (uint16_t*)p.h + from * p.ldh;
        f.ldy = p.ldh;
        f.act = p.act;
        return few(f, frags, st);
    };
    if (p.m <= few_limit(p.type)) {
        for (int64_t at = 0; at < p.m; at += FEW_ROWS)
            if ((rc = few_rows(at, p.m - at < FEW_ROWS ? p.m - at : FEW_ROWS))) return rc;
        return SPA_OK;
    }
    Operands o;
    if ((rc = operands(wk, run, p.type, p.gate, up, p.n, p.k, p.kind, p.x, p.m, p.ldx, false, o, st))) return rc;
    Gemm g = gemm_of(o, p.m, p.n);
    g.kind = p.kind;
    g.y = (uint16_t*)p.h;
    g.ldy = p.ldh;
    g.act = p.act;
    const int64_t tail = tail_rows(g, p.type);
    g.m -= (int)tail;
    if ((rc = multiply(g, wk, run, st))) return rc;
    return tail ? few_rows(p.m - tail, tail) : SPA_OK;
}

// grad = [dG | dU] in one matrix of 2 np columns; dx = grad [Wg; Wu] is then one product over 2 np, with the
// weights transposed side by side, and the weights' gradients are products over the rows. grad is rounded once to the
// operands' type, as a program that keeps it would store it: in float32 parts the products that follow would be twice
// or three times as many. BF16 holds any size; beside binary16 operands a power of two is taken out of each row, and for
// the weights' gradients (F16 weights) of each column in its place.
int gated_backward(const Gated& p, Work& wk, bool run, bool want_x, bool want_w, hipStream_t st) {
    int rc;
    const int64_t np = up64(p.n), mp = up64(p.m);
    Operands o;
    if ((rc = operands(wk, run, p.type, p.gate, run ? p.up : SOME, p.n, p.k, p.kind, p.x, p.m, p.ldx, true, o, st))) return rc;
    const int64_t wide = o.rest ? 4 * np : 2 * np, ldg = wide + PAD, ldm = mp + PAD;
    uint16_t* grad = wk.take<uint16_t>(p.m * ldg);
    int32_t *ge = nullptr, *ce = nullptr;                        // taken out of grad's rows; out of its columns
    if (o.norm) {
        ge = wk.take<int32_t>(p.m);
        void* top = wk.take<uint8_t>(8);
        if (run && (rc = grad_exponents((const uint16_t*)p.dh, p.kind, p.ldh, p.m, p.n, o.norm, o.n0, o.we0, o.n1, o.we1, top, ge, st)))
            return rc;
    } else if (o.half == SRC_F16) {
        ge = wk.take<int32_t>(p.m);
        ce = wk.take<int32_t>(2 * np);
        float *xn = wk.take<float>(p.m), *n0 = wk.take<float>(p.n), *n1 = wk.take<float>(p.n), *part = wk.take<float>(tops_part(p.m, p.n));
        if (run && (rc = norms16((const uint16_t*)p.x, p.ldx, p.m, (const uint16_t*)p.gate, (const uint16_t*)p.up, p.n, p.k, xn, n0, n1, st))) return rc;
        if (run && (rc = tops16((const uint16_t*)p.dh, p.ldh, p.m, p.n, xn, n0, n1, part, ge, ce, st))) return rc;
    }
    {
        Gemm g = gemm_of(o, p.m, p.n);
        g.kind = p.kind;
        g.act = p.act;
        g.dh = (const uint16_t*)p.dh;
        g.ldh = p.ldh;
        g.grad = grad;
        g.np = np;
        g.ldg = ldg;
        g.twice = o.rest != 0;
        g.ge = ge;
        if ((rc = multiply(g, wk, run, st))) return rc;
    }
    if (want_x) {
        uint16_t* wt = wk.take<uint16_t>(p.k * ldg);
        if (run && (rc = transpose16(o.w0, o.ldw, p.n, p.k, wt, ldg, np, nullptr, nullptr, st))) return rc;
        if (run && (rc = transpose16(o.w1, o.ldw, p.n, p.k, wt + np, ldg, np, nullptr, nullptr, st))) return rc;
        if (run && o.rest && (rc = transpose16(o.w0 + o.rest, o.ldw, p.n, p.k, wt + 2 * np, ldg, np, nullptr, nullptr, st))) return rc;
        if (run && o.rest && (rc = transpose16(o.w1 + o.rest, o.ldw, p.n, p.k, wt + 3 * np, ldg, np, nullptr, nullptr, st))) return rc;
        Gemm g{};
        g.half = o.half;
        g.x = grad;
        g.w0 = wt;
        g.ldx = g.ldw = ldg;
        g.m = (int)p.m;
        g.n = (int)p.k;
        g.k = (int)wide;
        g.xe = ge;
        g.kind = p.kind;
        g.y = (uint16_t*)p.dx;
        g.ldy = p.lddx;
        if ((rc = multiply(g, wk, run, st))) return rc;
    }
    if (want_w) {
        uint16_t* gt = wk.take<uint16_t>(2 * np * ldm);
        uint16_t* xt = wk.take<uint16_t>(p.k * ldm);
        if (run && (rc = transpose16(grad, ldg, p.m, 2 * np, gt, ldm, mp, ge, ce, st))) return rc;
        if (run && (rc = transpose16((const uint16_t*)p.x, p.ldx, p.m, p.k, xt, ldm, mp, nullptr, nullptr, st))) return rc;
        for (int i = 0; i < 2; ++i) {
            Gemm g{};
            g.half = o.half;
            g.x = gt + (i ? np * ldm : 0);
            g.w0 = xt;
            g.ldx = g.ldw = ldm;
            g.m = (int)p.n;
            g.n = (int)p.k;
            g.k = (int)mp;
            g.xe = ce ? ce + i * np : nullptr;
            g.kind = p.kind;
            g.y = (uint16_t*)(i ? p.dup : p.dgate);
            g.ldy = p.k;
            if ((rc = multiply(g, wk, run, st))) return rc;
        }
    }
    return SPA_OK;
}

}  // namespace
}  // namespace lin
}  // namespace spa

using namespace spa;
using namespace spa::lin;

extern "C" uint64_t spa_project_work_bytes(int type, int64_t n, int64_t k, int x_kind, int64_t m, int64_t pool, int64_t rank) {
    if (check_weight("", type, n, k) || check_rows("", x_kind, m, k, k) || pool < 0 || pool > INT32_MAX || (pool && (rank < 1 || rank > 256)) ||
        m == 0 || n == 0)
        return 0;
    Project p{};
    p.type = type, p.n = n, p.k = k, p.kind = x_kind, p.m = m, p.ldx = k, p.pool = pool, p.rank = rank;
    Work wk{nullptr};
    project(p, wk, false, nullptr);
    return wk.used;
}

extern "C" int spa_project(int type, const void* w, int64_t n, int64_t k, int x_kind, const void* x, int64_t m, int64_t x_stride,
                           void* y, int64_t y_stride, const void* a, const void* b, const float* scale, int64_t pool, int64_t rank,
                           const int32_t* which, void* work, uint64_t work_bytes, void* stream) {
    const char* who = "spa_project";
    int rc;
    if ((rc = check_weight(who, type, n, k)) || (rc = check_rows(who, x_kind, m, k, x_stride))) return rc;
    if (y_stride < n) return fail(SPA_ERR_ARG, "%s: output stride %lld for %lld columns", who, (long long)y_stride, (long long)n);
    if (pool < 0 || pool > INT32_MAX || (pool && (rank < 1 || rank > 256)))
        return fail(SPA_ERR_ARG, "%s: %lld adapters of rank %lld (1 to 256 are taken)", who, (long long)pool, (long long)rank);
    if (m == 0 || n == 0) return SPA_OK;
    if (!w || !x || !y || (pool && (!a || !b || !scale || !which))) return fail(SPA_ERR_ARG, "%s: null pointer", who);
    if (!on(x, 2) || !on(y, 2) || (pool && (!on(a, 2) || !on(b, 2) || !on(scale, 4) || !on(which, 4))))
        return fail(SPA_ERR_ARG, "%s: a pointer is not aligned to its elements", who);
    if ((rc = check_weight_at(who, type, w))) return rc;
    if ((rc = check_work(who, work, work_bytes, spa_project_work_bytes(type, n, k, x_kind, m, pool, rank)))) return rc;
    Work wk{(uint8_t*)work};
    return project(Project{type, w, n, k, x_kind, x, m, x_stride, y, y_stride, a, b, scale, pool, rank, which}, wk, true, (hipStream_t)stream);
}

namespace {
int check_act(const char* who, int act) {
    return act == ACT_SILU || act == ACT_GELU ? SPA_OK : fail(SPA_ERR_ARG, "%s: activation %d", who, act);
}
}  // namespace

extern "C" uint64_t spa_gated_work_bytes(int type, int64_t n, int64_t k, int x_kind, int64_t m) {
    if (check_weight("", type, n, k) || check_rows("", x_kind, m, k, k) || m == 0 || n == 0) return 0;
    Gated p{};
    p.type = type, p.n = n, p.k = k, p.kind = x_kind, p.m = m, p.ldx = k;
    Work wk{nullptr};
    gated(p, wk, false, nullptr);
    return wk.used;
}

extern "C" int spa_gated(int type, const void* gate, const void* up, int64_t n, int64_t k, int x_kind, const void* x, int64_t m,
                         int64_t x_stride, int act, void* h, int64_t h_stride, void* work, uint64_t work_bytes, void* stream) {
    const char* who = "spa_gated";
    int rc;
    if ((rc = check_weight(who, type, n, k)) || (rc = check_rows(who, x_kind, m, k, x_stride)) || (rc = check_act(who, act))) return rc;
    if (h_stride < n) return fail(SPA_ERR_ARG, "%s: output stride %lld for %lld columns", who, (long long)h_stride, (long long)n);
    if (m == 0 || n == 0) return SPA_OK;
    if (!gate || !up || !x || !h) return fail(SPA_ERR_ARG, "%s: null pointer", who);
    if (!on(x, 2) || !on(h, 2)) return fail(SPA_ERR_ARG, "%s: a pointer is not aligned to its elements", who);
    if ((rc = check_weight_at(who, type, gate)) || (rc = check_weight_at(who, type, up))) return rc;
    if ((rc = check_work(who, work, work_bytes, spa_gated_work_bytes(type, n, k, x_kind, m)))) return rc;
    Gated p{};
    p.type = type, p.gate = gate, p.up = up, p.n = n, p.k = k, p.kind = x_kind, p.x = x, p.m = m, p.ldx = x_stride, p.act = act;
    p.h = h, p.ldh = h_stride;
    Work wk{(uint8_t*)work};
    return gated(p, wk, true, (hipStream_t)stream);
}

extern "C" uint64_t spa_gated_backward_work_bytes(int type, int64_t n, int64_t k, int x_kind, int64_t m, int input_grad, int weight_grads) {
    if (check_weight("", type, n, k) || check_rows("", x_kind, m, k, k) || m == 0 || n == 0) return 0;
    Gated p{};
    p.type = type, p.n = n, p.k = k, p.kind = x_kind, p.m = m, p.ldx = k;
    Work wk{nullptr};
    gated_backward(p, wk, false, input_grad != 0, weight_grads != 0, nullptr);
    return wk.used;
}

extern "C" int spa_gated_backward(int type, const void* gate, const void* up, int64_t n, int64_t k, int x_kind, const void* x, int64_t m,
                                  int64_t x_stride, int act, const void* dh, int64_t dh_stride, void* dx, int64_t dx_stride,
                                  void* dgate, void* dup, void* work, uint64_t work_bytes, void* stream) {
    const char* who = "spa_gated_backward";
    int rc;
    if ((rc = check_weight(who, type, n, k)) || (rc = check_rows(who, x_kind, m, k, x_stride)) || (rc = check_act(who, act))) return rc;
    if (dh_stride < n || (dx && dx_stride < k)) return fail(SPA_ERR_ARG, "%s: stride %lld for %lld columns, %lld for %lld", who, (long long)dh_stride, (long long)n, (long long)dx_stride, (long long)k);
    if (!dgate != !dup) return fail(SPA_ERR_ARG, "%s: the gradient of one of the two matrices only", who);
    if (dgate && !(is16(type) && kind_of(type) == x_kind))
        return fail(SPA_ERR_TYPE, "%s: gradients of weights of type %d beside inputs of kind %d", who, type, x_kind);
    if (n > MOST_INNER || m > MOST_COLS) return fail(SPA_ERR_ARG, "%s: %lld rows, %lld weight rows are too many", who, (long long)m, (long long)n);
    if (!dx && !dgate) return SPA_OK;
    if (!on(x, 2) || !on(dh, 2) || !on(dx, 2) || !on(dgate, 2) || !on(dup, 2))
        return fail(SPA_ERR_ARG, "%s: a pointer is not aligned to its elements", who);
    hipStream_t st = (hipStream_t)stream;
    if (m == 0 || n == 0) {                                      // sums of nothing
        if (dx && m && (rc = zero_rows((uint16_t*)dx, dx_stride, m, k, st))) return rc;
        if (dgate && n && ((rc = zero_rows((uint16_t*)dgate, k, n, k, st)) || (rc = zero_rows((uint16_t*)dup, k, n, k, st)))) return rc;
        return SPA_OK;
    }
    if (!gate || !up || !x || !dh) return fail(SPA_ERR_ARG, "%s: null pointer", who);
    if ((rc = check_weight_at(who, type, gate)) || (rc = check_weight_at(who, type, up))) return rc;
    if ((rc = check_work(who, work, work_bytes, spa_gated_backward_work_bytes(type, n, k, x_kind, m, dx != nullptr, dgate != nullptr)))) return rc;
    Gated p{};
    p.type = type, p.gate = gate, p.up = up, p.n = n, p.k = k, p.kind = x_kind, p.x = x, p.m = m, p.ldx = x_stride, p.act = act;
    p.ldh = dh_stride, p.dh = dh, p.dx = dx, p.dgate = dgate, p.dup = dup, p.lddx = dx_stride;
    Work wk{(uint8_t*)work};
    return gated_backward(p, wk, true, dx != nullptr, dgate != nullptr, st);
}
