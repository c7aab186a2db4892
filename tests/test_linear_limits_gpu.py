"""The products with packed weights at the ends of their ranges, against float64 restatements: numbers that are not
finite and whom they may reach, the largest and the least inputs, and what the forms keep of weights of many bits.

Tolerances are those of test_linear_gpu (an output's rounding, K 2^-24 T for float32 sums of K terms, T the sum over
absolute values, and what a form's operands lose), with the operands' part named by each test."""
import numpy as np
import pytest

from seedpack_amd import linear
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
