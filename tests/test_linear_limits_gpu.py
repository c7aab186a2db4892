"""The products with packed weights at the ends of their ranges, against float64 restatements: numbers that are not
finite and whom they may reach, the largest and the least inputs, and what the forms keep of weights of many bits.

Tolerances are those of test_linear_gpu (an output's rounding, K 2^-24 T for float32 sums of K terms, T the sum over
absolute values, and what a form's operands lose), with the operands' part named by each test."""
import ctypes
import threading

import numpy as np
import pytest

from seedpack_amd import device as dev
from seedpack_amd import linear
from seedpack_amd._lib import LIB_PATH, check, lib
from seedpack_amd.gpuquant import GPUQuant
from seedpack_amd.requant import QFUN
from tests.test_linear_gpu import (BF16, F16, _named, adapters, close, gated_backward64, inputs, project64, random_blocks,  # noqa: F401
                                   rng, slack, store, up, weights, wide)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [BF16, F16])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("m,k,rank", [(40, 512, 5), (150, 512, 5), (300, 512, 16), (300, 2048, 20)])
def test_adapter_that_is_not_finite(m, k, rank, bad, kind):
    """one number of one adapter's second matrix: its own rows have what the definition says in that column; rows of
    other adapters and of none, in the same tile, are bit for bit as without it"""
    g = rng(40, m, k, kind is F16)
    n, pool = 140, 3
    w, w64 = weights(g, linear.F16 if kind is F16 else linear.BF16, n, k)
    x, x64 = inputs(g, m, k, kind)
    ad, a, b, s = adapters(g, pool, rank, n, k, kind)
    which = g.integers(-1, pool, m).astype(np.int32)
    clean = linear.project(up(x), w, ad, up(which)).to_host()
    worse = b.copy()
    worse[1, 9, 2] = bad
    got = linear.project(up(x), w, linear.Adapters(ad.a, up(store(worse, kind)), ad.scale), up(which)).to_host()
    mine = which == 1
    assert mine.any() and not mine.all()
    assert np.array_equal(got[~mine], clean[~mine])
    rest = np.arange(n) != 9
    y, total = project64(x64[mine], w64, a, b, s, which[mine])
    close(np.ascontiguousarray(got[mine][:, rest]), y[:, rest], slack(total[:, rest], k + rank), kind)
    want = bad * np.sign(x64[mine] @ a[1][2])
    assert np.array_equal(wide(got[mine][:, 9]), want, equal_nan=True)


@pytest.mark.parametrize("m", [1, 3, 20, 64, 100, 150])
@pytest.mark.parametrize("t", [linear.F16, linear.BF16, 2, 8, 12, 13, 14, 3, 16, 20, 23])
def test_project_largest_inputs(t, m):
    """BF16 inputs so large that the sums come near the largest float32 and codes times inputs pass it: finite as
    the definition is"""
    g = rng(41, t, m)
    n, k = 37, 512
    w, w64 = weights(g, t, n, k)
    x = g.normal(0, 1, (m, k))
    x *= 2.0 ** np.floor(np.log2(2.0 ** 127 / (np.abs(x) @ np.abs(w64.T)).max(1, keepdims=True)))
    x = store(np.clip(x, -3e38, 3e38), BF16)
    y, total = project64(wide(x), w64)
    assert total.max() < 3.4e38 and np.isfinite(wide(x)).all()
    close(linear.project(up(x), w).to_host(), y, slack(total, k), BF16)


@pytest.mark.parametrize("m", [1, 20, 64])
@pytest.mark.parametrize("t", [2, 8, 12, 13, 14])
def test_gated_largest_inputs(t, m):
    """the same gate beside an up projection of zeros: zeros, not an infinity times zero"""
    g = rng(42, t, m)
    n, k = 37, 512
    gate, w64 = weights(g, t, n, k)
    zero = linear.Weight(t, up(np.zeros(gate.data.nbytes, np.uint8)), n, k)
    x = g.normal(0, 1, (m, k))
    x *= 2.0 ** np.floor(np.log2(2.0 ** 127 / (np.abs(x) @ np.abs(w64.T)).max(1, keepdims=True)))
    assert (wide(linear.gated(up(store(np.clip(x, -3e38, 3e38), BF16)), gate, zero).to_host()) == 0).all()


@pytest.mark.parametrize("m", [1, 3, 40, 64])
@pytest.mark.parametrize("kind", [BF16, F16])
@pytest.mark.parametrize("t", [linear.F16, linear.BF16, 8, 12, 14, 10, 19])
def test_few_rows_with_numbers_that_are_not_finite(t, kind, m):
    """all of a row infinite or NaN, or one number in its first or last places: every output of the row as defined"""
    g = rng(43, t, m, kind is F16)
    n, k = 70, 1280
    w, w64 = weights(g, t, n, k)
    x, x64 = inputs(g, m, k, kind)
    clean = linear.project(up(x), w).to_host()
    for at, v in ((0, np.nan), (k - 1, np.nan), (slice(0, None), np.nan), (0, np.inf), (k - 1, -np.inf), (777, np.inf)):
        bad = x64.copy()
        bad[m // 2, at] = v
        got = linear.project(up(store(bad, kind)), w).to_host()
        keep = np.arange(m) != m // 2
        assert np.array_equal(got[keep], clean[keep])
        row = wide(got[m // 2])
        if np.isnan(v):
            assert np.isnan(row).all()
        else:
            with np.errstate(invalid="ignore"):
                assert np.array_equal(row, v * w64[:, at], equal_nan=True)


def backward_f16(g, m, n, k, sx, sw, sd):
    """F16 operands of the given sizes (powers of two), the columns of dh of unlike size -> what gated_backward takes, in float64 too"""
    pair = lambda shape, s: (lambda h: (h, wide(h)))(store(np.clip(g.normal(0, 1, shape) * s, -6e4, 6e4), F16))
    (x, x64), (wg, g64), (wu, u64) = pair((m, k), sx), pair((n, k), sw), pair((n, k), sw)
    dh, d64 = pair((m, n), sd * np.exp2(-g.integers(0, 9, n).astype(float)))
    return (x, wg, wu, dh), (x64, g64, u64, d64)


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("m,n,k", [(5, 64, 64), (150, 96, 70), (600, 300, 200)])
@pytest.mark.parametrize("sx,sw,sd,which", [(2.0 ** 5, 2.0 ** -8, 2.0 ** 14, ("dx",)), (2.0 ** -10, 2.0 ** 5, 2.0 ** 14, ("dgate", "dup")),
                                            (2.0 ** -16, 2.0 ** 8, 2.0 ** -16, ("dx",)), (2.0 ** 6, 2.0 ** -16, 2.0 ** -14, ("dgate", "dup"))])
def test_gated_backward_range(sx, sw, sd, which, m, n, k, act):
    """F16: inner gradients that pass the largest F16 number or fall below the least, and outputs that do not. Inner
    gradients are taken to 11 bits, and to 2^-34 of what their row (for dx; their column for the weights' gradients)
    can hold at most, 1.13 max |dh| |x| |w| (the powers of two put the bound between 2^11 and 2^15; half a step of F16 is 2^-25)"""
    g = rng(44, m, int(np.log2(sx)) + 50, len(act))
    (x, wg, wu, dh), (x64, g64, u64, d64) = backward_f16(g, m, n, k, sx, sw, sd)
    gate, upw = (linear.Weight(linear.F16, up(v), n, k) for v in (wg, wu))
    arrays = {"dx": np.zeros((m, k), F16), "dgate": np.zeros((n, k), F16), "dup": np.zeros((n, k), F16)}
    arrays = {name: up(a) for name, a in arrays.items()}
    linear.gated_backward(up(x), gate, upw, up(dh), act, **arrays)
    want = gated_backward64(x64, g64, u64, d64, act, k, 2.0 ** -11)
    xn, wn = np.linalg.norm(x64, axis=1), np.maximum(np.linalg.norm(g64, axis=1), np.linalg.norm(u64, axis=1))
    ad = np.abs(d64)
    # rows are held to their own bound before columns are to theirs: both parts for the weights' gradients
    rows = 2.0 ** -34 * 1.13 * ad.max(1) * xn * wn.max()
    cols = 2.0 ** -34 * 1.13 * (ad * xn[:, None]).max(0) * wn
    extra = {"dx": rows[:, None] * (np.abs(g64).sum(0) + np.abs(u64).sum(0))[None],
             "dgate": (rows @ np.abs(x64))[None] + cols[:, None] * np.abs(x64).sum(0)[None]}
    extra["dup"] = extra["dgate"]
    for name in which:
        y, off = want[name]
        assert 2.0 ** -14 < np.abs(y).max() < 60000, (name, np.abs(y).max())
        close(arrays[name].to_host(), y, off + extra[name], F16, name)


def test_gated_backward_rows_of_unlike_size():
    """F16 rows of dh and of x from far apart: each row of dx to its own size, the sums over rows to their largest"""
    g = rng(45)
    m, n, k = 200, 128, 96
    (x, wg, wu, dh), _ = backward_f16(g, m, n, k, 0.25, 0.05, 1.0)
    size = np.exp2(g.integers(-12, 12, (m, 1)).astype(float))
    dh = store(wide(dh) * size, F16)
    x64, g64, u64, d64 = wide(x), wide(wg), wide(wu), wide(dh)
    gate, upw = (linear.Weight(linear.F16, up(v), n, k) for v in (wg, wu))
    arrays = {"dx": up(np.zeros((m, k), F16)), "dgate": up(np.zeros((n, k), F16)), "dup": up(np.zeros((n, k), F16))}
    linear.gated_backward(up(x), gate, upw, up(dh), **arrays)
    want = gated_backward64(x64, g64, u64, d64, "silu", k, 2.0 ** -11)
    for name, a in arrays.items():
        close(a.to_host(), *want[name], F16, name)


@pytest.mark.parametrize("kind", [BF16, F16])
@pytest.mark.parametrize("m", [20, 150])
@pytest.mark.parametrize("t", [8, 12, 14])
def test_blocks_of_large_scales_and_no_weights(t, m, kind):
    """a block whose scale is the largest and whose codes (or their scales) are zero, beside blocks of tiny weights:
    the tiny ones count in full"""
    g = rng(46, t, m, kind is F16)
    n, k = 50, 512
    _, qk, bs = QFUN[t]
    b, _ = random_blocks(g, t, n, k)
    b = b.reshape(n, k // qk, bs)
    at = {8: [0], 12: [0, 2], 14: [208]}[t]
    for o in at:
        b[:, :, o:o + 2] = np.frombuffer(np.float16(2.0 ** -20).tobytes(), np.uint8)
    codes = slice(2, 34) if t == 8 else (slice(4, 16) if t == 12 else slice(192, 208))
    if t == 12:
        b[:, :, 4:16] = 0x11 * g.integers(0, 2, b[:, :, 4:16].shape, dtype=np.uint8)      # scales and offsets 0, 1, 16, 17
    elif t == 14:
        b[:, :, codes] = 1
    else:
        b[:, :, codes] = g.integers(0, 3, b[:, :, codes].shape, dtype=np.uint8)
    b[:, 0, at[0]:at[0] + 2] = np.frombuffer(np.float16(65504).tobytes(), np.uint8)
    b[:, 0, codes] = 0
    w64 = GPUQuant().dequantize(t, b.reshape(-1), k).to_host().reshape(n, k).astype(np.float64)
    assert (w64[:, :qk] <= 0).all() and np.abs(w64).max() < 1e-2
    w64[:, :qk] += 0.0
    x, x64 = inputs(g, m, k, kind)
    y, total = project64(x64, w64)
    scale = 1.0 if kind is BF16 else 2.0 ** 10       # F16 outputs: away from its least numbers
    if kind is F16:
        x, x64 = store(x64 * scale, kind), x64 * scale
        y, total = project64(wide(x), w64)
    close(linear.project(up(x), linear.Weight(t, up(b.reshape(-1)), n, k)).to_host(), y,
          slack(total, k, 2.0 ** -11 if kind is BF16 else 2.0 ** -21), kind)


@pytest.mark.parametrize("t", [2, 8, 12, 14, 23])
def test_long_rows_of_blocks(t):
    """rows of more weights than the conversion to binary16 holds at once, their largest weight in the last part"""
    g = rng(52, t)
    n, k, m = 9, 16384 + 512, 140
    b, _ = random_blocks(g, t, n, k)
    _, qk, bs = QFUN[t]
    b = b.reshape(n, k // qk, bs)
    at = {14: 208}.get(t, 0)
    b[:, -1, at:at + 2] = np.frombuffer(np.float16(0.25).tobytes(), np.uint8)
    w64 = GPUQuant().dequantize(t, b.reshape(-1), k).to_host().reshape(n, k).astype(np.float64)
    x, x64 = inputs(g, m, k, BF16)
    y, total = project64(x64, w64)
    close(linear.project(up(x), linear.Weight(t, up(b.reshape(-1)), n, k)).to_host(), y, slack(total, k), BF16)


def near_pairs(g, values, count):
    """pairs of (index, index) of values that round to the same 11 bits and differ by 2^-11.5 of themselves or more, the first the larger"""
    v = np.asarray(values, np.float64)
    e = np.exp2(np.floor(np.log2(v)))
    held = np.round(v / e * 1024) / 1024 * e              # to 11 bits
    out = []
    for i in g.permutation(len(v)):
        j = np.flatnonzero((held == held[i]) & (v < v[i] * (1 - 2.0 ** -11.5)))
        if len(j):
            out.append((i, int(g.choice(j))))
            if len(out) == count:
                return out
    raise AssertionError("too few pairs")


def fine_blocks(g, t, n, k):
    """n rows whose runs of 32 weights are +v1 and -v2 in turn, v1 and v2 the same 11-bit number but not the same -> bytes, weights"""
    _, qk, bs = QFUN[t]
    b = np.zeros((n, k // qk, bs), np.uint8)
    put = lambda r, j, o, h: b[r, j].__setitem__(slice(o, o + 2), np.frombuffer(np.float16(h).tobytes(), np.uint8))
    d = (1024 + np.arange(1024)) * 2.0 ** -19             # all F16 numbers of one binary order
    if t in (6, 8):
        # Q8_0: codes 64..127 and their negatives; Q5_0: 8..15 (its codes are held over 16)
        q = np.arange(64, 128) if t == 8 else np.arange(8, 16)
        pairs = near_pairs(g, (d[:, None] * q).reshape(-1), n * k // 64)
        for i, (a, c) in enumerate(pairs):
            r, j = divmod(i, k // 64)
            for s, p in ((0, a), (1, c)):
                put(r, 2 * j + s, 0, d[p // len(q)])
                code = int(q[p % len(q)]) * (1 - 2 * s)
                if t == 8:
                    b[r, 2 * j + s, 2:] = code & 0xff
                else:
                    b[r, 2 * j + s, 2:6] = 0xff if code + 16 >= 16 else 0
                    b[r, 2 * j + s, 6:] = ((code + 16) & 15) * 0x11
    else:                                                 # Q4_K: d sc 15 and -dm mn, 32 weights each
        for r in range(n):
            while True:
                a, c = int(g.integers(1024)), int(g.integers(1024))
                sc, mn = np.meshgrid(np.arange(32, 64), np.arange(32, 64), indexing="ij")
                v1, v2 = d[a] * sc * 15, 16 * d[c] * mn
                e = np.exp2(np.floor(np.log2(v1)))
                ok = np.argwhere((np.round(v1 / e * 1024) == np.round(v2 / e * 1024)) & (v1 * (1 - 2.0 ** -11.5) > v2))
                if len(ok):
                    i, j = ok[g.integers(len(ok))]
                    break
            s, o = np.zeros(8, int), np.zeros(8, int)
            s[::2], o[1::2] = 32 + i, 32 + j
            for blk in range(k // qk):
                put(r, blk, 0, d[a])
                put(r, blk, 2, 16 * d[c])
                b[r, blk, 4:8] = s[:4] | (s[4:] >> 4 << 6)
                b[r, blk, 8:12] = o[:4] | (o[4:] >> 4 << 6)
                b[r, blk, 12:16] = (s[4:] & 15) | ((o[4:] & 15) << 4)
                b[r, blk, 16:] = 0x0f                     # the even runs' codes 15, the odd runs' 0
    w = GPUQuant().dequantize(t, b.reshape(-1), k).to_host().reshape(n, k).astype(np.float64)
    assert (w.reshape(n, -1, 2, 32)[:, :, 0] > 0).all() and (w.reshape(n, -1, 2, 32)[:, :, 1] < 0).all()
    return b.reshape(-1), w


@pytest.mark.parametrize("t,kind,m,extra", [(8, F16, 3, 0), (8, F16, 40, 0), (12, F16, 3, 0), (12, F16, 40, 0), (8, BF16, 3, 0), (8, BF16, 40, 0), (12, BF16, 3, 0), (12, BF16, 40, 0),
                                            (6, F16, 3, 2.0 ** -16), (6, F16, 40, 2.0 ** -16), (6, BF16, 3, 2.0 ** -16), (6, BF16, 40, 2.0 ** -16),
                                            (8, F16, 150, 2.0 ** -21), (6, F16, 150, 2.0 ** -21), (12, F16, 150, 2.0 ** -21), (12, F16, 700, 2.0 ** -21)])
def test_weights_beyond_eleven_bits(t, kind, m, extra):
    """weights whose first 11 bits cancel: what is left are the bits beyond. Few rows of Q8_0 and Q4_K go by codes (Q4_K's
    beside BF16 as 128 + code), whose sums of 32 are added one after another: (32 + k / 32) roundings, of sums so many
    times T (an offset of Q4_K is that of 15 codes in each of 32 terms, and no more than T)"""
    g = rng(47, t, m, kind is F16)
    n, k = 60, 256 if t == 12 else 64
    b, w64 = fine_blocks(g, t, n, k)
    x = g.random((m, k // 64, 1, 32)) + 0.5
    x = store(np.broadcast_to(x, (m, k // 64, 2, 32)).reshape(m, k), kind)
    y, total = project64(wide(x), w64)
    per = {(8, F16): 1, (8, BF16): 1, (12, F16): 2, (12, BF16): 2 * 143 / 15}.get((t, kind)) if m <= 128 else None
    allowed = total * ((per * (32 + k / 32) if per else k) * 2.0 ** -24 + extra)
    assert (np.abs(y) > 2.0 ** -12.6 * total).all() and (allowed < 0.4 * np.abs(y)).all()
    close(linear.project(up(x), linear.Weight(t, up(b), n, k)).to_host(), y, allowed, kind)


@pytest.mark.parametrize("t", [8, 12])
@pytest.mark.parametrize("m", [20, 300])
def test_gradient_through_weights_beyond_eleven_bits(t, m):
    """the same for the inputs' gradient: rows of the gate in pairs of +v1 and -v2, gates of zero (silu' = 1/2, silu = 0), up
    projections of one power of two"""
    g = rng(48, t, m)
    n, k = 64, 256
    _, qk, bs = QFUN[t]
    fine, _ = fine_blocks(g, t, n, 64 if t == 8 else 256)
    rows = fine.reshape(n, -1, bs)
    gate = np.zeros((n, k // qk, bs), np.uint8)
    if t == 8:                                            # run 0 of a fine row into all of row 2 i, run 1 into 2 i + 1
        for i in range(n // 2):
            gate[2 * i], gate[2 * i + 1] = rows[i, 0], rows[i, 1]
        upw = np.zeros((n, k // qk, bs), np.uint8)
        upw[:, :, :2] = np.frombuffer(np.float16(2.0 ** -12).tobytes(), np.uint8)
        upw[:, ::2, 2:], upw[:, 1::2, 2:] = 64, 0xc0
    else:                                                 # all runs d sc 15, or all -dm mn
        gate[:n] = rows[:n]
        for i in range(n // 2):
            gate[2 * i] = gate[2 * i + 1] = rows[i, 0]
            sc, mn = int(rows[i, 0, 4] & 63), int(rows[i, 0, 9] & 63)
            for r, s, o in ((2 * i, sc, 0), (2 * i + 1, 0, mn)):
                gate[r, :, 4:8], gate[r, :, 8:12] = s | (s >> 4 << 6), o | (o >> 4 << 6)
                gate[r, :, 12:16] = (s & 15) | ((o & 15) << 4)
                gate[r, :, 16:] = 0xff if s else 0
        upw = np.zeros((n, k // qk, bs), np.uint8)
        for o in (0, 2):
            upw[:, :, o:o + 2] = np.frombuffer(np.float16(2.0 ** -8).tobytes(), np.uint8)
        s, o = np.zeros(8, int), np.zeros(8, int)
        s[::2], o[1::2] = 1, 8
        upw[:, :, 4:8], upw[:, :, 8:12] = s[:4], o[:4]
        upw[:, :, 12:16] = (s[4:] & 15) | ((o[4:] & 15) << 4)
        upw[:, :, 16:] = 0x08                             # 8 in the even runs, 0 in the odd
    of = lambda b: GPUQuant().dequantize(t, b.reshape(-1), k).to_host().reshape(n, k).astype(np.float64)
    g64, u64 = of(gate), of(upw)
    x64 = np.broadcast_to(np.where(np.arange(k) // 32 % 2, -1.0, 1.0), (m, k))
    assert not (x64 @ g64.T).any() and len(np.unique(np.abs(u64))) == 1 and (g64[::2] > 0).all() and (g64[1::2] < 0).all()
    u = x64 @ u64.T
    assert (u == u[0, 0]).all() and u[0, 0] > 0
    d64 = np.repeat(np.exp2(g.integers(-4, 3, (m, n // 2)).astype(float)), 2, axis=1)
    dg = 0.5 * d64 * u
    y, total = dg @ g64, np.abs(dg) @ np.abs(g64)
    allowed = total * (2 * n * 2.0 ** -24 + 2.0 ** -21)
    assert (y > 0.4 * 2.0 ** -13 * total).all() and (allowed < 0.2 * y).all()
    wt = lambda b: linear.Weight(t, up(b.reshape(-1)), n, k)
    dx = linear.gated_backward(up(store(x64, F16)), wt(gate), wt(upw), up(store(d64, F16)))[0]
    close(dx.to_host(), y, allowed, F16)


@pytest.mark.parametrize("t,kind", [(linear.BF16, BF16), (linear.F16, F16)])
@pytest.mark.parametrize("m", [1, 20, 150, 1100])
def test_products_of_one_type_are_exact(t, kind, m):
    """operands of one 16-bit type: nothing but the float32 sums and the output's rounding"""
    g = rng(49, m, t)
    n, k = 133, 192
    w, w64 = weights(g, t, n, k)
    x, x64 = inputs(g, m, k, kind)
    y, total = project64(x64, w64)
    close(linear.project(up(x), w).to_host(), y, slack(total, k, 0), kind)


@pytest.mark.parametrize("kind", [BF16, F16])
@pytest.mark.parametrize("m,pool,rank", [(1, 40, 256), (20, 40, 3), (64, 100, 17), (100, 40, 16), (150, 3, 256), (300, 33, 200)])
def test_adapters_of_large_pools_and_ranks(m, pool, rank, kind):
    """more adapters than a tile has rows, ranks up to the largest"""
    g = rng(51, m, rank, kind is F16)
    n, k = 70, 256
    w, w64 = weights(g, 12, n, k)
    x, x64 = inputs(g, m, k, kind)
    ad, a, b, s = adapters(g, pool, rank, n, k, kind)
    which = g.integers(-1, pool + 1, m).astype(np.int32)
    which[0] = pool - 1
    y, total = project64(x64, w64, a, b, s, which)
    close(linear.project(up(x), w, ad, up(which)).to_host(), y, slack(total, k + rank), kind)


@pytest.mark.parametrize("kind", [BF16, F16])
@pytest.mark.parametrize("t", [8, 12, linear.F16])
@pytest.mark.parametrize("m", [64, 65, 100, 128, 129])
def test_adapters_first_product_over_a_long_k(t, m, kind):
    """rows around the number from which all adapters' first products are one product; their order is any"""
    g = rng(55, t, m, kind is F16)
    n, k, pool, rank = 70, 4096, 5, 20
    w, w64 = weights(g, t, n, k)
    x, x64 = inputs(g, m, k, kind)
    ad, a, b, s = adapters(g, pool, rank, n, k, kind)
    which = g.integers(-1, pool + 1, m).astype(np.int32)
    y, total = project64(x64, w64, a, b, s, which)
    close(linear.project(up(x), w, ad, up(which)).to_host(), y, slack(total, k + rank), kind)


def test_streams_that_end():
    """workspaces of streams that come and go: right results, and release() afterwards"""
    g = rng(53)
    n, k, m = 300, 1024, 140
    w, w64 = weights(g, 12, n, k)
    x, x64 = inputs(g, m, k, BF16)
    y, total = project64(x64, w64)
    xd = up(x)
    for _ in range(6):
        st = dev.Stream()
        out = linear.project(xd, w, stream=st.handle)
        close(out.to_host(stream=st.handle), y, slack(total, k), BF16)
        del out, st
    linear.release()
    close(linear.project(xd, w).to_host(), y, slack(total, k), BF16)


def test_threads_at_once():
    """two threads, each with a stream of its own, many and few rows in turn: every result as alone"""
    g = rng(56)
    n, k = 300, 1024
    w, _ = weights(g, 12, n, k)
    x = {m: inputs(g, m, k, BF16)[0] for m in (3, 140, 300)}
    want = {m: linear.project(up(a), w).to_host() for m, a in x.items()}
    wrong = []

    def work():
        st = dev.Stream()
        arrays = {m: dev.DeviceArray.from_host(a, st.handle) for m, a in x.items()}
        for _ in range(8):
            got = {m: linear.project(a, w, stream=st.handle) for m, a in arrays.items()}
            wrong.extend(m for m, a in got.items() if not np.array_equal(a.to_host(stream=st.handle), want[m]))
        linear.release()

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


class Graph:
    """what a stream's calls left in a capture, by the HIP runtime that the library is linked with"""

    def __init__(self, stream, calls):
        self.hip = ctypes.CDLL(LIB_PATH)
        graph, self.made = ctypes.c_void_p(), ctypes.c_void_p()
        self.ok(self.hip.hipStreamBeginCapture(ctypes.c_void_p(stream), 0))
        try:
            calls()
        finally:
            self.ok(self.hip.hipStreamEndCapture(ctypes.c_void_p(stream), ctypes.byref(graph)))
        self.ok(self.hip.hipGraphInstantiate(ctypes.byref(self.made), graph, None, None, ctypes.c_size_t(0)))
        self.ok(self.hip.hipGraphDestroy(graph))

    def ok(self, code):
        assert code == 0, code

    def replay(self, stream):
        self.ok(self.hip.hipGraphLaunch(self.made, ctypes.c_void_p(stream)))

    def close(self):
        self.ok(self.hip.hipGraphExecDestroy(self.made))


@pytest.mark.parametrize("t", [linear.BF16, 8, 10])
@pytest.mark.parametrize("m", [1, 20, 300])
def test_captured_calls(t, m):
    """all four calls in one graph, replayed on new numbers between eager calls: the same bits; a captured call without
    its own memory is refused, and the graph's memory is not what eager calls use"""
    g = rng(54, t, m)
    n, k = 512, 2048
    (gate, _), (upw, _) = weights(g, t, n, k), weights(g, t, n, k)
    pool = adapters(g, 3, 16, n, k, BF16)[0]
    ids = up(g.integers(-1, 4, m).astype(np.int32))
    x, dh, work = (dev.DeviceArray(s, d) for s, d in (((m, k), BF16), ((m, n), BF16), (1 << 26, np.uint8)))
    outs = {"y": ((m, n), BF16), "h": ((m, n), BF16), "dx": ((m, k), BF16), "sums": ((1, k), np.float32), "counts": (1, np.int64)}
    if t == linear.BF16:
        outs |= {"dgate": ((n, k), BF16), "dup": ((n, k), BF16)}
    outs = {name: dev.DeviceArray(*of) for name, of in outs.items()}
    st = dev.Stream()

    def calls(**memory):
        linear.project(x, gate, pool, ids, out=outs["y"], stream=st.handle, **memory)
        linear.gated(x, gate, upw, out=outs["h"], stream=st.handle, **memory)
        linear.gated_backward(x, gate, upw, dh, stream=st.handle, **{d: outs[d] for d in ("dx", "dgate", "dup") if d in outs}, **memory)
        linear.add_squares(x, outs["sums"], outs["counts"], stream=st.handle, **memory)

    def captured():
        calls(work=work)
        with pytest.raises(ValueError):
            linear.gated(x, gate, upw, stream=st.handle, work=work)
        with pytest.raises(ValueError):
            linear.gated_backward(x, gate, upw, dh, dx=outs["dx"], stream=st.handle)

    def clear():
        outs["sums"].zero(st.handle)
        outs["counts"].zero(st.handle)

    def result():
        st.synchronize()
        return {name: a.to_host(stream=st.handle).tobytes() for name, a in outs.items()}

    calls(work=work)
    st.synchronize()
    graph = Graph(st.handle, captured)
    for _ in range(4):
        for a in (x, dh):
            h = store(g.normal(0, 0.3, a.shape), BF16)
            check(lib().spa_memcpy_h2d(a.ptr, h.ctypes.data, h.nbytes, st.handle))
        clear()
        graph.replay(st.handle)
        got = result()
        clear()
        calls()
        assert got == result()
    graph.close()
