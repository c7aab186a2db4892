"""The products with packed weights against float64 restatements (numpy, on the host).

Tolerances, derived from the arithmetic. Every output is a float32 sum rounded once to its 16-bit type, so it
is within u |y| + d of the exact value y (u = 2^-8 for BF16 with its 8 significant bits, 2^-11 for F16; half
of that is the rounding itself), where d is what the operands' forms and the float32 sums lose: with T the
same sum over absolute values, float32 adds of K terms lose at most K 2^-24 T in any order, and weights taken
to 11 bits (16 where rows are few) 2^-11 T (their rounding, and the rows' powers of two lose nothing). Each
test names its own d as a multiple of T."""
import sys

import numpy as np
import pytest

from seedpack_amd import device as dev
from seedpack_amd import linear
from seedpack_amd._lib import SpaError
from seedpack_amd.gpuquant import GPUQuant
from seedpack_amd.requant import NAMES, QFUN

pytestmark = pytest.mark.gpu

BF16, F16 = np.uint16, np.float16
UNIT = {BF16: 2.0 ** -8, F16: 2.0 ** -11}


@pytest.fixture(autouse=True)
def _named(request):
    print(request.node.name, file=sys.stderr, flush=True)


def rng(*key):
    return np.random.Generator(np.random.PCG64(list(key)))


def store(v, kind):
    """float64 -> the bits of a 16-bit type, to nearest even"""
    if kind is F16:
        return v.astype(np.float16)
    f = v.astype(np.float32)
    b = f.view(np.uint32)
    r = ((b.astype(np.uint64) + 0x7fff + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isfinite(f), r, (b >> 16).astype(np.uint16) | np.isnan(f) * np.uint16(0x40)).astype(np.uint16)


def wide(a):
    if a.dtype == np.float16:
        return a.astype(np.float64)
    return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def up(a):
    return dev.DeviceArray.from_host(np.ascontiguousarray(a))


def random_blocks(g, t, n, k, scale=True):
    """n rows of random blocks of a type with scales of real size -> (bytes, float64 weights by the dequantizer,
    which equals the reference's bit for bit)"""
    _, qk, bs = QFUN[t]
    b = g.integers(0, 256, (n * k // qk, bs), dtype=np.uint8)
    at = {2: [0], 3: [0, 2], 6: [0], 7: [0, 2], 8: [0], 10: [80, 82], 11: [108], 12: [0, 2], 13: [0, 2], 14: [208],
          16: [0], 17: [0], 18: [0], 19: [0], 20: [0], 21: [0], 22: [0], 23: [0], 42: [0]}.get(t, [])
    for o in at:
        d = (g.random(len(b)) * 4e-3 + 1e-4).astype(np.float16)
        b[:, o:o + 2] = d.view(np.uint8).reshape(-1, 2)
    if t == 29:                                    # the scale's 16 bits in the high nibbles of four words
        d = (g.random(len(b)) * 4e-3 + 1e-4).astype(np.float16).view(np.uint16)
        for i in range(4):
            b[:, 49 + 2 * i] = (b[:, 49 + 2 * i] & 0x0f) | (((d >> (4 * i)) & 15) << 4).astype(np.uint8)
    w = GPUQuant().dequantize(t, b.reshape(-1), k).to_host().reshape(n, k).astype(np.float64)
    return b.reshape(-1), w


def weights(g, t, n, k):
    """-> (Weight, float64 weights)"""
    if t in (linear.F16, linear.BF16):
        h = store(g.normal(0, 0.02, (n, k)), F16 if t == linear.F16 else BF16)
        return linear.Weight(t, up(h), n, k), wide(h)
    b, w = random_blocks(g, t, n, k)
    return linear.Weight(t, up(b), n, k), w


def inputs(g, m, k, kind):
    x = store(g.normal(0, 1, (m, k)) * np.exp(g.normal(0, 0.5, k)), kind)
    return x, wide(x)


def close(got, want, slack, kind, what=""):
    got = wide(got)
    off = np.abs(got - want) - (UNIT[kind] * np.abs(want) + slack + (2.0 ** -24 if kind is F16 else 0))
    assert got.shape == want.shape and not (off > 0).any(), (what, float(off.max()), np.argwhere(off > 0)[:4].tolist())
    assert np.isfinite(got).all()


def project64(x, w, a=None, b=None, scale=None, which=None):
    """-> (y, the same over absolute values)"""
    y, t = x @ w.T, np.abs(x) @ np.abs(w.T)
    if a is not None:
        for r, i in enumerate(which):
            if 0 <= i < len(scale):
                y[r] += float(scale[i]) * (b[i] @ (a[i] @ x[r]))
                t[r] += abs(float(scale[i])) * (np.abs(b[i]) @ (np.abs(a[i]) @ np.abs(x[r])))
    return y, t


def slack(t, k, extra=2.0 ** -11):
    return t * (k * 2.0 ** -24 + extra)


def adapters(g, count, rank, n, k, kind):
    a, b = store(g.normal(0, 1, (count, rank, k)) / np.sqrt(k), kind), store(g.normal(0, 0.1, (count, n, rank)), kind)
    s = (g.random(count) + 0.5).astype(np.float32)
    return linear.Adapters(up(a), up(b), up(s)), wide(a), wide(b), s


@pytest.mark.parametrize("kind", [BF16, F16])
@pytest.mark.parametrize("t", [linear.F16, linear.BF16] + sorted(QFUN))
def test_project_types(t, kind):
    """every type of weights, with few and with many rows, an odd number of outputs"""
    g = rng(1, t, kind is F16)
    n, k = 133, 768
    w, w64 = weights(g, t, n, k)
    for m in (1, 3, 33, 65, 130):
        x, x64 = inputs(g, m, k, kind)
        y, total = project64(x64, w64)
        close(linear.project(up(x), w).to_host(), y, slack(total, k), kind, (t, m))


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 127, 128, 129, 200, 257])
@pytest.mark.parametrize("t,kind", [(linear.BF16, BF16), (12, BF16), (8, F16)])
def test_project_rows(t, kind, m):
    g = rng(2, t, m)
    n, k = 257, 512
    w, w64 = weights(g, t, n, k)
    x, x64 = inputs(g, m, k, kind)
    y, total = project64(x64, w64)
    close(linear.project(up(x), w).to_host(), y, slack(total, k), kind)


@pytest.mark.parametrize("n,k", [(1, 1), (3, 7), (16, 31), (17, 33), (64, 63), (65, 65), (31, 100), (200, 1001), (5, 4096 + 8)])
@pytest.mark.parametrize("m", [1, 5, 70])
def test_project_odd_sizes(n, k, m):
    """16-bit weights take any number of columns"""
    for t, kind in ((linear.BF16, BF16), (linear.F16, F16), (linear.F16, BF16), (linear.BF16, F16)):
        g = rng(3, n, k, m, t)
        w, w64 = weights(g, t, n, k)
        x, x64 = inputs(g, m, k, kind)
        y, total = project64(x64, w64)
        close(linear.project(up(x), w).to_host(), y, slack(total, k), kind, (t, kind))


@pytest.mark.parametrize("rank", [1, 5, 8, 16, 24, 64, 100])
@pytest.mark.parametrize("m", [1, 7, 64, 65, 300])
@pytest.mark.parametrize("t,kind", [(12, BF16), (linear.F16, F16), (linear.BF16, BF16)])
def test_project_adapters(t, kind, m, rank):
    """rows of many adapters in any order, rows without one, numbers outside the pool"""
    g = rng(4, t, m, rank)
    n, k, pool = 130, 512, 5
    w, w64 = weights(g, t, n, k)
    x, x64 = inputs(g, m, k, kind)
    ad, a, b, s = adapters(g, pool, rank, n, k, kind)
    which = g.choice(np.array([-7, -1, 0, 1, 2, 3, 4, 5, 2 ** 31 - 1], np.int32), m)
    which[-1] = 4
    y, total = project64(x64, w64, a, b, s, which)
    got = linear.project(up(x), w, ad, up(which)).to_host()
    close(got, y, slack(total, k + rank), kind)


def test_project_adapter_alone():
    """weights of zero: what is left is the adapters' part alone, to the same bound"""
    g = rng(5)
    n, k, m, rank = 96, 256, 90, 16
    for kind in (BF16, F16):
        w = linear.Weight(linear.F16 if kind is F16 else linear.BF16, up(np.zeros((n, k), np.uint16)), n, k)
        x, x64 = inputs(g, m, k, kind)
        ad, a, b, s = adapters(g, 3, rank, n, k, kind)
        which = g.integers(0, 3, m).astype(np.int32)
        y, total = project64(x64, np.zeros((n, k)), a, b, s, which)
        for rows in (m, 20):
            close(linear.project(up(x[:rows]), w, ad, up(which[:rows])).to_host(), y[:rows],
                  slack(total[:rows], k, 2.0 ** -15), kind)


@pytest.mark.parametrize("m", [3, 70])
def test_project_strides_and_offsets(m):
    """rows further apart than their columns, arrays that begin at any element, blocks at any byte; what lies
    between the rows of the output stays"""
    g = rng(6, m)
    n, k, pool = 45, 256, 2
    for t, kind in ((12, BF16), (14, F16), (8, BF16), (linear.BF16, BF16)):
        for xo, ldx, yo, ldy, wo in ((0, k, 0, n, 0), (8, k + 8, 4, n + 3, 2), (1, k + 5, 3, n + 1, 7), (3, k, 1, n, 1)):
            if t == linear.BF16:
                wo = 0
            w, w64 = weights(g, t, n, k)
            x, x64 = inputs(g, m, k, kind)
            wide_x = np.full(xo + m * ldx, np.nan, np.float32).astype(F16) if kind is F16 else np.full(xo + m * ldx, 0x7fc0, BF16)
            for r in range(m):
                wide_x[xo + r * ldx:xo + r * ldx + k] = x[r]
            xd = up(wide_x)
            out0 = g.integers(0, 1 << 16, yo + m * ldy + 9).astype(np.uint16)
            od = up(out0)
            raw = np.concatenate([np.full(wo, 0xff, np.uint8), w.data.to_host().view(np.uint8).reshape(-1)])
            wd = up(raw)
            wv = linear.Weight(t, wd.view(wo, (len(raw) - wo,), np.uint8), n, k)
            ad, a, b, s = adapters(g, pool, 8, n, k, kind)
            which = g.integers(-1, pool, m).astype(np.int32)
            y, total = project64(x64, w64, a, b, s, which)
            linear.project(dev.DeviceArray((m, k), kind, ptr=xd.ptr + 2 * xo, owner=xd), wv, ad, up(which),
                           out=dev.DeviceArray((m, n), kind, ptr=od.ptr + 2 * yo, owner=od), x_stride=ldx, out_stride=ldy)
            got = od.to_host()
            rows = np.stack([got[yo + r * ldy:yo + r * ldy + n] for r in range(m)]).view(kind)
            close(rows, y, slack(total, k), kind, (t, xo, ldx, yo, ldy, wo))
            keep = np.ones(len(got), bool)
            for r in range(m):
                keep[yo + r * ldy:yo + r * ldy + n] = False
            assert np.array_equal(got[keep], out0[keep])


@pytest.mark.parametrize("m", [2, 80])
def test_project_unlike_sizes(m):
    """rows of very unlike size, weights whose blocks are far apart in size, the least and largest numbers: the
    powers of two that the many-rows form takes out lose nothing"""
    g = rng(7, m)
    n, k = 70, 512
    x = store(g.normal(0, 1, (m, k)) * np.exp2(g.integers(-60, 60, (m, 1)).astype(float)), BF16)
    b, _ = random_blocks(g, 8, n, k)
    blocks = b.reshape(n, -1, 34)
    d = np.exp2(g.integers(-20, 9, (n, 1)) + g.integers(-3, 1, (n, k // 32)).astype(float)).astype(np.float16)
    blocks[:, :, :2] = d.view(np.uint8).reshape(n, -1, 2)
    w64 = GPUQuant().dequantize(8, blocks.reshape(-1), k).to_host().reshape(n, k).astype(np.float64)
    y, total = project64(wide(x), w64)
    close(linear.project(up(x), linear.Weight(8, up(blocks.reshape(-1)), n, k)).to_host(), y, slack(total, k), BF16)


@pytest.mark.parametrize("m", [4, 72])
def test_project_infinite_and_nan_rows(m):
    """a row with an infinity or NaN gives what the definition gives, the others are as without it"""
    g = rng(8, m)
    n, k = 40, 256
    for t in (linear.BF16, 12):
        w, w64 = weights(g, t, n, k)
        x, x64 = inputs(g, m, k, BF16)
        clean = linear.project(up(x), w).to_host()
        bad = x.copy()
        bad[1, 5], bad[2, 9] = 0x7f80, 0x7fc0
        got = linear.project(up(bad), w).to_host()
        keep = np.arange(m) > 2
        keep[0] = True
        assert np.array_equal(got[keep], clean[keep])
        assert np.isnan(wide(got[2])).all()
        sure = np.abs(w64[:, 5]) > 0
        assert np.array_equal(wide(got[1])[sure], np.where(w64[:, 5] > 0, np.inf, -np.inf)[sure])



def same_class(got, want, sure, what):
    """infinities and NaN where the definition has them"""
    got = wide(got)
    odd = sure & ~np.isfinite(want)
    ok = np.where(np.isnan(want), np.isnan(got), got == want) | ~odd
    assert odd.any() and ok.all(), (what, np.argwhere(~ok)[:4].tolist())


@pytest.mark.parametrize("kind", [BF16, F16])
@pytest.mark.parametrize("t", [linear.F16, linear.BF16] + sorted(QFUN))
def test_project_infinities_of_every_type(t, kind):
    """one infinity in a row, and two that cancel: what the weights in front of them make of it, whatever form they
    take (weights below 2^-30 of their row's largest, which the many-rows form may take as zero, are left out)"""
    g = rng(30, t, kind is F16)
    n, k = 37, 256
    w, w64 = weights(g, t, n, k)
    fit = (np.abs(w64) >= 2.0 ** -30 * np.abs(w64).max(1, keepdims=True)) | (w64 == 0)
    for m in (3, 40, 150):
        x, x64 = inputs(g, m, k, kind)
        x64[0, 7], x64[1, 100], x64[2, 31], x64[2, 200] = np.inf, -np.inf, np.inf, np.inf
        with np.errstate(invalid="ignore"):
            want = np.stack([np.where(np.isinf(x64[r]), x64[r] * w64, 0).sum(1) for r in range(3)])
        sure = np.stack([fit[:, np.isinf(x64[r])].all(1) for r in range(3)])
        got = linear.project(up(store(x64, kind)), w).to_host()
        same_class(got[:3], want, sure, (t, m))
        assert np.isfinite(wide(got[3:])).all()


@pytest.mark.parametrize("kind", [BF16, F16])
@pytest.mark.parametrize("m,k", [(3, 512), (40, 512), (150, 512), (300, 2048)])
def test_adapters_infinite_inputs(m, k, kind):
    """an infinite input's part by way of an adapter of rank one, beside the projection's own; other rows as without"""
    g = rng(31, m, kind is F16)
    n = 70
    w, w64 = weights(g, linear.F16 if kind is F16 else linear.BF16, n, k)
    pool, a64, b64, s = adapters(g, 3, 1, n, k, kind)
    which = g.integers(0, 3, m).astype(np.int32)
    x, x64 = inputs(g, m, k, kind)
    clean = linear.project(up(x), w, pool, up(which)).to_host()
    x64[1, 9] = -np.inf
    i = which[1]
    with np.errstate(invalid="ignore"):
        want = -np.inf * w64[:, 9] + s[i] * b64[i][:, 0] * (-np.inf * a64[i][0, 9])
    got = linear.project(up(store(x64, kind)), w, pool, up(which)).to_host()
    same_class(got[1], want, np.ones(n, bool), (m, k))
    keep = np.arange(m) != 1
    assert np.array_equal(got[keep], clean[keep])


def act64(g, act):
    t = g if act == "silu" else 2 * np.sqrt(2 / np.pi) * (g + 0.044715 * g ** 3)
    dt = np.ones_like(g) if act == "silu" else 2 * np.sqrt(2 / np.pi) * (1 + 3 * 0.044715 * g ** 2)
    with np.errstate(over="ignore"):
        p, q = 1 / (1 + np.exp(-t)), 1 / (1 + np.exp(t))
    return g * p, p + g * p * q * dt


def gated64(x, wg, wu, act, k):
    """-> (h, a bound on what errors of g and u within slack() do to it)"""
    g, u = x @ wg.T, x @ wu.T
    tg, tu = slack(np.abs(x) @ np.abs(wg.T), k), slack(np.abs(x) @ np.abs(wu.T), k)
    v, _ = act64(g, act)
    # |act'| <= 1.13; the activation itself to 2^-20 of its value (expf and one division)
    return v * u, np.abs(u) * (1.13 * tg) + np.abs(v) * tu + 1.13 * tg * tu + 2.0 ** -20 * np.abs(v * u)


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("t,kind", [(linear.BF16, BF16), (linear.F16, F16), (linear.F16, BF16)] +
                         [(t, BF16) for t in sorted(QFUN)] + [(12, F16), (16, F16)])
def test_gated(t, kind, act):
    g = rng(10, t, kind is F16, len(act))
    n, k = 150, 512
    gate, g64 = weights(g, t, n, k)
    upw, u64 = weights(g, t, n, k)
    for m in (1, 19, 40, 66, 140):
        x, x64 = inputs(g, m, k, kind)
        h, off = gated64(x64, g64, u64, act, k)
        close(linear.gated(up(x), gate, upw, act).to_host(), h, off, kind, m)


@pytest.mark.parametrize("n,k,m", [(1, 1, 1), (7, 33, 3), (33, 100, 70), (64, 64, 64), (129, 65, 129), (1000, 129, 300)])
def test_gated_odd_sizes(n, k, m):
    for t, kind in ((linear.BF16, BF16), (linear.F16, F16)):
        g = rng(11, n, k, m)
        gate, g64 = weights(g, t, n, k)
        upw, u64 = weights(g, t, n, k)
        x, x64 = inputs(g, m, k, kind)
        h, off = gated64(x64, g64, u64, "silu", k)
        close(linear.gated(up(x), gate, upw).to_host(), h, off, kind)


@pytest.mark.parametrize("m", [2, 70])
def test_gated_far_arguments(m):
    """gates far to either side: the activation's limits, not NaN"""
    k = 64
    for v in (1e4, -1e4, 3e18, -3e18, 100.0, -100.0):
        x = store(np.full((m, k), v / k), BF16)
        one = linear.Weight(linear.BF16, up(store(np.ones((16, k)), BF16)), 16, k)
        for act in ("silu", "gelu"):
            h = wide(linear.gated(up(x), one, one, act).to_host())
            s = wide(x)[0].sum()
            want = max(s, 0.0) * s if abs(s) > 1e3 or act == "gelu" else s * s / (1 + np.exp(-s))
            assert np.allclose(h, want, rtol=2.0 ** -7, atol=1e-30), (v, act, h[0, 0], want)


def gated_backward64(x, wg, wu, dh, act, k, unit):
    """-> {name: (gradient, bound)}: g and u as in gated64, dG and dU rounded once to `unit`"""
    ax, ag, au, ad = np.abs(x), np.abs(wg), np.abs(wu), np.abs(dh)
    n, m = len(wg), len(x)
    g, u = x @ wg.T, x @ wu.T
    tg, tu = slack(ax @ ag.T, k), slack(ax @ au.T, k)
    v, d = act64(g, act)
    dg, du = dh * u * d, dh * v
    # act'' is at most 1.2 in size for both activations (silu'' <= 1/2, gelu'' <= 2 sqrt(2/pi) / sqrt(2))
    og = ad * (np.abs(d) * tu + (np.abs(u) + tu) * 1.2 * tg) + (unit + 2.0 ** -20) * np.abs(dg)
    ou = ad * 1.13 * tg + (unit + 2.0 ** -20) * np.abs(du)
    adg, adu = np.abs(dg) + og, np.abs(du) + ou
    sums = lambda a, b, kk: slack(a @ b, kk)
    return {"dx": (dg @ wg + du @ wu, og @ ag + ou @ au + sums(adg, ag, 2 * n) + sums(adu, au, 2 * n)),
            "dgate": (dg.T @ x, og.T @ ax + sums(adg.T, ax, m)),
            "dup": (du.T @ x, ou.T @ ax + sums(adu.T, ax, m))}


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("n,k,m", [(1, 1, 1), (50, 40, 3), (130, 70, 65), (256, 256, 64), (300, 129, 150), (65, 520, 33)])
def test_gated_backward(n, k, m, act):
    for t, kind in ((linear.BF16, BF16), (linear.F16, F16)):
        g = rng(12, n, k, m)
        gate, g64 = weights(g, t, n, k)
        upw, u64 = weights(g, t, n, k)
        x, x64 = inputs(g, m, k, kind)
        dh = store(g.normal(0, 0.1, (m, n)) * np.exp(g.normal(0, 1, (m, 1))), kind)
        want = gated_backward64(x64, g64, u64, wide(dh), act, k, UNIT[kind])
        small = 0 if kind is BF16 else 2.0 ** -24         # F16 inner gradients: steps of 2^-24 near zero
        extra = {"dx": small * (np.abs(g64).sum(0) + np.abs(u64).sum(0))[None], "dgate": small * np.abs(x64).sum(0)[None],
                 "dup": small * np.abs(x64).sum(0)[None]}
        arrays = {"dx": dev.DeviceArray((m, k), kind), "dgate": dev.DeviceArray((n, k), kind), "dup": dev.DeviceArray((n, k), kind)}
        linear.gated_backward(up(x), gate, upw, up(dh), act, **arrays)
        for name, a in arrays.items():
            close(a.to_host(), want[name][0], want[name][1] + extra[name], kind, name)
        dx, dgate, _ = linear.gated_backward(up(x), gate, upw, up(dh), act)
        assert dgate is None and np.array_equal(dx.to_host(), arrays["dx"].to_host())
        dx, dgate, dup = linear.gated_backward(up(x), gate, upw, up(dh), act, dgate=dev.DeviceArray((n, k), kind), dup=dev.DeviceArray((n, k), kind))
        assert dx is None and np.array_equal(dgate.to_host(), arrays["dgate"].to_host())
        assert np.array_equal(dup.to_host(), arrays["dup"].to_host())


@pytest.mark.parametrize("t,kind", [(t, BF16) for t in sorted(QFUN)] + [(12, F16), (linear.F16, BF16), (linear.BF16, F16)])
def test_gated_backward_frozen(t, kind):
    """the gradient of the inputs through weights of another type: inner gradients to 11 bits, rows of unlike size"""
    g = rng(13, t, kind is F16)
    n, k, m = 90, 256, 70
    gate, g64 = weights(g, t, n, k)
    upw, u64 = weights(g, t, n, k)
    x, x64 = inputs(g, m, k, kind)
    size = np.exp2(g.integers(-24, 10, (m, 1)).astype(float)) if kind is BF16 else 1.0
    dh = store(g.normal(0, 0.1, (m, n)) * size, kind)
    want, off = gated_backward64(x64, g64, u64, wide(dh), "silu", k, 2.0 ** -11)["dx"]
    # and each inner gradient to 2^-20 of its row's bound: 1.13 |dh|max |x| |w|max
    top = max(np.linalg.norm(g64, axis=1).max(), np.linalg.norm(u64, axis=1).max())
    floor = 2.0 ** -20 * 1.13 * np.abs(wide(dh)).max(1) * np.linalg.norm(x64, axis=1) * top
    off = off + floor[:, None] * (np.abs(g64).sum(0) + np.abs(u64).sum(0))[None]
    dx, _, _ = linear.gated_backward(up(x), gate, upw, up(dh))
    close(dx.to_host(), want, off, kind)


def test_gated_backward_against_differences():
    """the gradient along random directions against central differences of the float64 forward pass"""
    g = rng(14)
    n, k, m = 96, 64, 40
    for act in ("silu", "gelu"):
        gate, g64 = weights(g, linear.BF16, n, k)
        upw, u64 = weights(g, linear.BF16, n, k)
        x, x64 = inputs(g, m, k, BF16)
        dh = store(g.normal(0, 1, (m, n)), BF16)
        arrays = {"dx": dev.DeviceArray((m, k), BF16), "dgate": dev.DeviceArray((n, k), BF16), "dup": dev.DeviceArray((n, k), BF16)}
        linear.gated_backward(up(x), gate, upw, up(dh), act, **arrays)
        loss = lambda a, b, c: float((wide(dh) * act64(a @ b.T, act)[0] * (a @ c.T)).sum())
        e = 1e-5
        for name, at in (("dx", 0), ("dgate", 1), ("dup", 2)):
            base = [x64, g64, u64]
            d = g.normal(0, 1, base[at].shape)
            hi = loss(*[v + e * d if i == at else v for i, v in enumerate(base)])
            lo = loss(*[v - e * d if i == at else v for i, v in enumerate(base)])
            got = wide(arrays[name].to_host())
            slope = float((got * d).sum())
            # outputs and inner gradients each to 2^-8, independent over the entries; the difference to e^2
            bound = 2.0 ** -7 * np.sqrt(((got * d) ** 2).sum()) + 2.0 ** -8 * abs(slope) + 1e-4 * (1 + abs(slope))
            assert abs((hi - lo) / (2 * e) - slope) <= 4 * bound, (act, name, (hi - lo) / (2 * e), slope)


def test_gated_backward_strides_and_nothing():
    g = rng(15)
    n, k, m = 37, 48, 9
    gate, g64 = weights(g, linear.BF16, n, k)
    upw, u64 = weights(g, linear.BF16, n, k)
    x, x64 = inputs(g, m, k, BF16)
    dh = store(g.normal(0, 1, (m, n)), BF16)
    want = linear.gated_backward(up(x), gate, upw, up(dh))[0].to_host()
    wide_x, wide_d = np.full((m, k + 3), 0x7fc0, BF16), np.full((m, n + 1), 0x7fc0, BF16)
    wide_x[:, :k], wide_d[:, :n] = x, dh
    xd, dd, od = up(wide_x), up(wide_d), up(np.full((m, k + 7), 0x1234, BF16))
    linear.gated_backward(dev.DeviceArray((m, k), BF16, ptr=xd.ptr, owner=xd), gate, upw, dev.DeviceArray((m, n), BF16, ptr=dd.ptr, owner=dd),
                          dx=dev.DeviceArray((m, k), BF16, ptr=od.ptr, owner=od), x_stride=k + 3, dh_stride=n + 1, dx_stride=k + 7)
    got = od.to_host()
    assert np.array_equal(got[:, :k], want) and (got[:, k:] == 0x1234).all()
    # no rows: the weights' gradients are zero
    dgate, dup = up(np.full((n, k), 0x7fc0, BF16)), up(np.full((n, k), 0x7fc0, BF16))
    linear.gated_backward(dev.DeviceArray((0, k), BF16), gate, upw, dev.DeviceArray((0, n), BF16), dgate=dgate, dup=dup,
                          dx=dev.DeviceArray((0, k), BF16))
    assert not dgate.to_host().any() and not dup.to_host().any()
    assert linear.project(dev.DeviceArray((0, k), BF16), gate).shape == (0, n)
    assert linear.gated(dev.DeviceArray((0, k), BF16), gate, upw).shape == (0, n)



@pytest.mark.parametrize("t,kind", [(linear.BF16, BF16), (linear.F16, F16), (8, BF16), (8, F16), (12, F16)])
@pytest.mark.parametrize("m", [3, 300])
def test_gated_backward_infinite_gradient(t, kind, m):
    """an infinity in one row of dh: that row of dx is what the weights make of it, the others are as without it"""
    g = rng(32, t, kind is F16, m)
    n, k = 96, 256
    (gate, wg), (up_, wu) = weights(g, t, n, k), weights(g, t, n, k)
    x, x64 = inputs(g, m, k, kind)
    d64 = wide(store(g.normal(0, 1, (m, n)), kind))
    clean = linear.gated_backward(up(x), gate, up_, up(store(d64, kind)))[0].to_host()
    d64[1, 17] = np.inf
    gv, uv = x64[1] @ wg[17], x64[1] @ wu[17]
    value, slope = act64(gv, "silu")
    with np.errstate(invalid="ignore"):
        want = np.inf * (uv * slope) * wg[17] + np.inf * value * wu[17]
    got = linear.gated_backward(up(x), gate, up_, up(store(d64, kind)))[0].to_host()
    sure = np.ones(k, bool)
    for w in (wg[17], wu[17]):
        sure &= (np.abs(w) >= 2.0 ** -20 * np.abs(w).max()) | (w == 0)
    same_class(got[1], want, sure, (t, m))
    keep = np.arange(m) != 1
    assert np.array_equal(got[keep], clean[keep])


@pytest.mark.parametrize("kind", [BF16, F16, np.float32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 513), (7, 100), (33, 511), (512, 520), (2000, 33), (1025, 1024)])
def test_add_squares(rows, cols, kind):
    """float32 sums of at most a few thousand squares: within rows 2^-24 of the exact sum"""
    g = rng(20, rows, cols)
    x = g.normal(0, 1, (rows, cols)) * np.exp(g.normal(0, 1, cols))
    x = x.astype(np.float32) if kind is np.float32 else store(x, kind)
    x64 = x.astype(np.float64) if kind is np.float32 else wide(x)
    sums0 = g.random((1, cols)).astype(np.float32)
    sums, counts = up(sums0), up(np.array([5], np.int64))
    linear.add_squares(up(x), sums, counts)
    want = sums0 + (x64 ** 2).sum(0)
    assert (np.abs(sums.to_host() - want) <= want * (rows + 4) * 2.0 ** -24).all()
    assert counts.to_host()[0] == 5 + rows


@pytest.mark.parametrize("rows,cols,experts,each", [(1, 5, 3, 1), (100, 600, 7, 2), (2500, 130, 64, 2), (3000, 520, 2, 3), (50, 64, 300, 1)])
def test_add_squares_experts(rows, cols, experts, each):
    """rows of several experts, of one twice, of none; experts without a row keep their sums"""
    g = rng(21, rows, cols, experts)
    x = store(g.normal(0, 1, (rows, cols)), BF16)
    which = g.integers(-1, experts + 1, (rows, each)).astype(np.int32)
    which[which == experts // 2] = -1
    which[0] = 0
    sums0 = g.random((experts, cols)).astype(np.float32)
    sums, counts = up(sums0), up(np.arange(experts, dtype=np.int64))
    linear.add_squares(up(x), sums, counts, up(which))
    want, n = sums0.astype(np.float64), np.arange(experts)
    for r in range(rows):
        for e in which[r]:
            if 0 <= e < experts:
                want[e] += wide(x[r]) ** 2
                n[e] += 1
    got = sums.to_host()
    assert np.array_equal(counts.to_host(), n)
    assert (np.abs(got - want) <= want * (rows + 4) * 2.0 ** -24).all()
    none = n == np.arange(experts)
    assert none.any() and np.array_equal(got[none], sums0[none])
    again = up(sums0)
    linear.add_squares(up(x), again, up(np.arange(experts, dtype=np.int64)), up(which))
    assert np.array_equal(again.to_host(), got)


def test_add_squares_strides():
    g = rng(22)
    for kind, off, ld in ((BF16, 1, 77), (BF16, 8, 80), (np.float32, 3, 71), (F16, 0, 72)):
        x = g.normal(0, 1, (40, 70))
        x = x.astype(np.float32) if kind is np.float32 else store(x, kind)
        raw = np.full(off + 40 * ld, 0x7fc0, BF16) if kind is BF16 else np.full(off + 40 * ld, np.nan, kind)
        for r in range(40):
            raw[off + r * ld:off + r * ld + 70] = x[r]
        d = up(raw)
        sums, counts = up(np.zeros((1, 70), np.float32)), up(np.zeros(1, np.int64))
        linear.add_squares(dev.DeviceArray((40, 70), kind, ptr=d.ptr + off * raw.itemsize, owner=d), sums, counts, x_stride=ld)
        want = ((x.astype(np.float64) if kind is np.float32 else wide(x)) ** 2).sum(0)
        assert (np.abs(sums.to_host()[0] - want) <= want * 44 * 2.0 ** -24).all()


def test_add_squares_gathers_an_importance():
    """squares -> imatrix -> quantizer: the same blocks as with the importance made on the host"""
    g = rng(23)
    x, x64 = inputs(g, 300, 512, BF16)
    sums, counts = up(np.zeros((1, 512), np.float32)), up(np.zeros(1, np.int64))
    for r in range(0, 300, 100):
        linear.add_squares(up(x[r:r + 100]), sums, counts)
    imx = (sums.to_host()[0] / np.float32(counts.to_host()[0])).astype(np.float32)
    assert np.allclose(imx, (x64 ** 2).mean(0), rtol=1e-5)
    w = store(g.normal(0, 0.02, (64, 512)), BF16)
    blocks = GPUQuant().quantize_tensors(12, [(w.reshape(-1), 512)], [imx], device=True)[0]
    q64 = GPUQuant().dequantize(12, blocks, 512).to_host().reshape(64, 512).astype(np.float64)
    y, total = project64(x64[:70], q64)
    close(linear.project(up(x[:70]), linear.Weight(12, blocks, 64, 512)).to_host(), y, slack(total, 512), BF16)


@pytest.mark.parametrize("m,n,k", [(4100, 2100, 192), (2100, 4100, 128), (300, 2053, 1024), (700, 130, 2112)])
@pytest.mark.parametrize("t,kind", [(linear.BF16, BF16), (8, BF16), (8, F16)])
def test_project_tiles(t, kind, m, n, k):
    """enough outputs for the large tiles, and few enough for pieces of k; both ragged, with adapters"""
    g = rng(31, t, m)
    w, w64 = weights(g, t, n, k)
    x, x64 = inputs(g, m, k, kind)
    ad, a, b, s = adapters(g, 3, 20, n, k, kind)
    which = np.sort(g.integers(-1, 3, m)).astype(np.int32)
    y, total = x64 @ w64.T, np.abs(x64) @ np.abs(w64.T)
    for i in range(3):
        at = which == i
        y[at] += float(s[i]) * ((x64[at] @ a[i].T) @ b[i].T)
        total[at] += float(s[i]) * ((np.abs(x64[at]) @ np.abs(a[i].T)) @ np.abs(b[i].T))
    close(linear.project(up(x), w, ad, up(which)).to_host(), y, slack(total, k + 20), kind)
    y, total = project64(x64, w64)
    close(linear.project(up(x), w).to_host(), y, slack(total, k), kind)


@pytest.mark.parametrize("m,n,k", [(2100, 2060, 128), (300, 700, 1024), (150, 200, 2048)])
@pytest.mark.parametrize("t,kind", [(linear.BF16, BF16), (12, BF16)])
def test_gated_tiles(t, kind, m, n, k):
    g = rng(32, t, m)
    k = -(-k // 256) * 256 if t == 12 else k
    gate, g64 = weights(g, t, n, k)
    upw, u64 = weights(g, t, n, k)
    x, x64 = inputs(g, m, k, kind)
    h, off = gated64(x64, g64, u64, "silu", k)
    close(linear.gated(up(x), gate, upw).to_host(), h, off, kind)
    dh = store(g.normal(0, 0.1, (m, n)), kind)
    want, off = gated_backward64(x64, g64, u64, wide(dh), "silu", k, UNIT[BF16] if t == linear.BF16 else 2.0 ** -11)["dx"]
    if t == 12:
        top = max(np.linalg.norm(g64, axis=1).max(), np.linalg.norm(u64, axis=1).max())
        floor = 2.0 ** -20 * 1.13 * np.abs(wide(dh)).max(1) * np.linalg.norm(x64, axis=1) * top
        off = off + floor[:, None] * (np.abs(g64).sum(0) + np.abs(u64).sum(0))[None]
    close(linear.gated_backward(up(x), gate, upw, up(dh))[0].to_host(), want, off, kind)


def test_project_last_rows_and_long_adapters():
    """five rows beyond whole tiles, which the few-rows form takes, and adapters' first products as one product:
    all of the last rows and a sample of the others, a sample of the columns"""
    g = rng(33)
    m, n, k, pool, rank = 2053, 4096, 12288, 4, 64
    b, w64 = random_blocks(g, 12, 256, k)                 # 16 times the same 256 rows
    w = linear.Weight(12, up(np.tile(b, 16)), n, k)
    x, x64 = inputs(g, m, k, BF16)
    ad, a, bb, s = adapters(g, pool, rank, n, k, BF16)
    which = np.sort(g.integers(-1, pool, m)).astype(np.int32)
    rows = np.concatenate([np.arange(0, m - 16, 97), np.arange(m - 16, m)])
    cols = np.arange(0, n, 37)
    y, total = project64(x64[rows], w64[cols % 256], a, bb[:, cols], s, which[rows])
    got = linear.project(up(x), w, ad, up(which)).to_host()
    close(np.ascontiguousarray(got[rows][:, cols]), y, slack(total, k + rank), BF16)


def test_streams_and_repeats():
    """work on a stream of its own; the same call twice gives the same bits"""
    g = rng(30)
    n, k = 300, 1024
    w, _ = weights(g, 12, n, k)
    st = dev.Stream()
    for m in (3, 90):
        x, _ = inputs(g, m, k, BF16)
        xd = dev.DeviceArray.from_host(x, st.handle)
        a = linear.project(xd, w, stream=st.handle)
        b = linear.project(xd, w, stream=st.handle)
        st.synchronize()
        assert np.array_equal(a.to_host(stream=st.handle), b.to_host(stream=st.handle))


def test_refusals_on_device():
    x = up(np.zeros((4, 256), BF16))
    w = linear.Weight(12, up(np.zeros(8 * 144, np.uint8)), 8, 256)
    with pytest.raises(SpaError):                       # 16-bit weights off their alignment
        raw = up(np.zeros(8 * 256 + 1, BF16))
        linear.project(x, linear.Weight(linear.BF16, dev.DeviceArray(8 * 256, BF16, ptr=raw.ptr + 2, owner=raw), 8, 256))
    with pytest.raises(SpaError):                       # a workspace that is too small
        linear.project(up(np.zeros((100, 256), BF16)), w, work=dev.DeviceArray(256, np.uint8))
    with pytest.raises(SpaError):                       # weight gradients of blocks
        linear.gated_backward(x, w, w, up(np.zeros((4, 8), BF16)), dgate=dev.DeviceArray((8, 256), BF16), dup=dev.DeviceArray((8, 256), BF16))
