"""Routing to experts and the join of their results against float64 restatements.

Tolerances, derived from the arithmetic. u is half a step of the result's type, relative to the value.
  weights: ratios taken in float64 (logarithms up to 1000, so to 2^-36 at the least) and rounded once to float32. Softmax without renorm divides
    by a float32 sum of up to 1024 terms: each term's expf is off by a step of 2^-23 and by the rounding of l - max, whose size d
    costs d 2^-24 of a term e^-d, at most 2^-25 of the largest; 16 terms a lane and 6 joins lose 22 2^-24. 32 2^-24 in all.
  logits' gradient: a sum of at most 33 float32 terms (one expert's places, and the share of the row's sum), each as exact as a
    weight: (32 + 33 + 3) 2^-24 of their magnitudes' sum t, and u of the value.
  join: `each` float32 terms, each one rounding by fma: each 2^-24 t, and u. dy: one float32 product and u. dweights: n
    products and adds in some order, n 2^-24 t."""
import sys
import threading

import numpy as np
import pytest

from seedpack_amd import device as dev
from seedpack_amd import experts
from seedpack_amd._lib import SpaError, check, lib

from . import experts_oracle as oracle
from .experts_oracle import BF16, F16, F32, HALF, LEAST, rng, store, wide

pytestmark = pytest.mark.gpu
KINDS = [BF16, F16, F32]


@pytest.fixture(autouse=True)
def _named(request):
    print(request.node.name, file=sys.stderr, flush=True)


def up(a):
    return dev.DeviceArray.from_host(np.ascontiguousarray(a))


def close(got, want, t, kind):
    """got within t of want, and its own rounding"""
    got = wide(got)
    room = t + HALF[kind] * (abs(want) + t) + LEAST[kind]
    bad = ~(abs(got - want) <= room)
    assert not bad.any(), (int(bad.sum()), got[bad][:4], want[bad][:4], (abs(got - want) / room)[bad][:4])


def check_route(l, each, score, renorm=True, scale=1.0, bias=None, stride=None, **groups):
    """l: the logits in their type"""
    m, e = l.shape
    x = up(l)
    if stride:
        h = np.full((m, stride), 7, l.dtype)
        h[:, :e] = l
        base = up(h)
        x = dev.DeviceArray((m, e), l.dtype, ptr=base.ptr, owner=base)
    r = experts.route(x, each, score, None if bias is None else up(bias), renorm=renorm, scale=scale, logits_stride=stride, **groups)
    v = wide(l)
    want = oracle.choose(v, each, score, bias, **groups)
    which = r.which.to_host()
    np.testing.assert_array_equal(which, want)
    w = oracle.weights(v, want, score, renorm, scale)
    close(r.weights.to_host(), w, (2.0 ** -36 if renorm or score == "sigmoid" else 32 * 2.0 ** -24) * abs(w), F32)
    order, starts = oracle.by_expert(want, e)
    np.testing.assert_array_equal(r.starts.to_host(), starts)
    np.testing.assert_array_equal(r.order.to_host(), order)
    return which


SIZES = [(1, 1, 1), (1, 8, 2), (3, 64, 8), (65, 65, 3), (130, 128, 8), (1, 256, 8), (257, 256, 16), (33, 257, 32), (5, 512, 1), (70, 1024, 32),
         (4099, 60, 4), (20, 17, 17)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("score,renorm", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
@pytest.mark.parametrize("rows,e,each", SIZES)
def test_route(rows, e, each, score, renorm, kind):
    g = rng(1, rows, e, each)
    check_route(store(g.normal(0, 2, (rows, e)), kind), each, score, renorm, 2.5)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("rows,e,each,groups,keep,best", [(50, 256, 8, 8, 4, 2), (7, 160, 6, 8, 3, 1), (40, 66, 5, 3, 2, 2), (9, 64, 3, 64, 5, 2),
                                                          (11, 1024, 32, 16, 3, 2), (300, 12, 2, 2, 1, 2), (33, 200, 4, 40, 7, 1)])
@pytest.mark.parametrize("biased", [False, True])
def test_route_groups_and_bias(rows, e, each, groups, keep, best, biased, score, kind):
    g = rng(2, rows, e, groups)
    bias = g.normal(0, 0.1, e).astype(F32) if biased else None
    check_route(store(g.normal(0, 1, (rows, e)), kind), each, score, bias=bias, groups=groups, keep=keep, best=best)


@pytest.mark.parametrize("rows", [64, 65, 4096, 4097, 4500])
@pytest.mark.parametrize("e,each,groups", [(64, 32, 8), (65, 5, 5), (128, 32, 4), (129, 8, 3), (256, 32, 64), (257, 9, 1), (512, 3, 16), (1024, 32, 64)])
@pytest.mark.parametrize("kind", KINDS)
def test_route_by_few_and_many_lanes(kind, e, each, groups, rows):
    """each number of lanes a row, of a lane's experts and of a workgroup's rows, whole and partly masked, with ties"""
    g = rng(10, rows, e)
    l = store(g.normal(0, 1, (rows, e)), kind)
    l[g.random(l.shape) < 0.2] = store(np.array([-np.inf]), kind)[0]
    l[::9] = store(np.array([-np.inf]), kind)[0]
    l[::7, ::3] = store(np.array([0.5]), kind)[0]
    bias = g.normal(0, 0.2, e).astype(F32)
    check_route(l, each, "softmax", renorm=False)
    check_route(l, each, "sigmoid", scale=1.5)
    check_route(l, each, "sigmoid", bias=bias)
    if groups > 1:
        least = -(-each * groups // e)
        check_route(l, each, "softmax", bias=bias, groups=groups, keep=min(groups, least + 1), best=2)
        check_route(l, each, "sigmoid", groups=groups, keep=least, best=1)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_bias_alone(score):
    g = rng(3)
    check_route(g.normal(0, 1, (513, 100)).astype(F32), 7, score, bias=g.normal(0, 0.3, 100).astype(F32))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_route_ties_and_masks(biased, score, kind):
    """equal logits, zeros of both signs, the type's lowest value, -inf: ties to the lowest number, -inf never"""
    g = rng(4, biased)
    l = g.integers(-2, 3, (64, 48)).astype(np.float64)
    l[3] = 0
    l[4] = np.where(np.arange(48) % 2, 0.0, -0.0)
    l[5] = -np.inf
    l[6, 2:] = -np.inf                               # two left, four asked for
    low = {BF16: -3.3895313892515355e38, F16: -65504.0, F32: -3.4028234663852886e38}[kind]
    l[7] = low
    l[8, 1:] = low
    l[9] = -900                                      # scores that vanish together
    l[10] = np.where(np.arange(48) < 40, -np.inf, -800 - np.arange(48))
    which = check_route(store(l, kind), 4, score, bias=np.zeros(48, F32) if biased else None)
    assert (which[5] == -1).all() and list(which[6] >= 0) == [True, True, False, False]


def test_route_groups_with_masked_experts():
    g = rng(5)
    l = g.normal(0, 1, (40, 32)).astype(F32)
    l[0] = -np.inf
    l[1, 8:] = -np.inf
    l[2, ::2] = -np.inf
    l[3, 1:] = -np.inf
    check_route(l, 6, "sigmoid", bias=g.normal(0, 0.1, 32).astype(F32), groups=4, keep=2)
    check_route(l, 6, "softmax", groups=4, keep=2, best=1)


def test_route_bias_of_minus_infinity_masks():
    l = rng(6).normal(0, 1, (20, 16)).astype(F32)
    bias = np.zeros(16, F32)
    bias[::2] = -np.inf
    r = experts.route(up(l), 10, "sigmoid", up(bias))
    which = r.which.to_host()
    assert (which[:, 8:] == -1).all() and (which[:, :8] % 2 == 1).all() and (r.weights.to_host()[:, 8:] == 0).all()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_not_a_number(score):
    """a NaN is above all and reaches its row's weights only"""
    l = rng(7).normal(0, 1, (6, 40)).astype(F32)
    l[2, 17] = l[2, 30] = np.nan
    l[4, 3] = -np.nan
    r = experts.route(up(l), 3, score)
    which, w = r.which.to_host(), r.weights.to_host()
    assert list(which[2][:2]) == [17, 30] and which[4][0] == 3 and np.isnan(w[[2, 4]]).all()
    keep = [0, 1, 3, 5]
    np.testing.assert_array_equal(which[keep], oracle.choose(wide(l[keep]), 3, score))
    assert np.isfinite(w[keep]).all()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_not_a_number_in_a_group(score):
    """a group with a NaN and nothing beside it is above all, and no more than `keep` groups are kept"""
    l = rng(20).normal(0, 1, (3, 24)).astype(F32)
    l[1, 4:8] = np.nan, -np.inf, -np.inf, -np.inf
    which = experts.route(up(l), 4, score, groups=6, keep=1).which.to_host()
    if score == "sigmoid":                           # with softmax all of the row's scores are NaN
        assert list(which[1]) == [4, -1, -1, -1]
    assert (which[1] < 8).all()
    np.testing.assert_array_equal(which[[0, 2]], oracle.choose(wide(l[[0, 2]]), 4, score, groups=6, keep=1))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("e,stride", [(64, 72), (64, 65), (130, 136), (5, 5)])
def test_route_strides(e, stride, kind):
    check_route(store(rng(8, e).normal(0, 1, (77, e)), kind), 4, "softmax", stride=stride)


def test_route_without_rows():
    r = experts.route(dev.DeviceArray((0, 16), F32), 4)
    assert r.which.shape == (0, 4) and (r.starts.to_host() == 0).all()
    assert experts.route_backward(dev.DeviceArray((0, 16), F32), r.which, dev.DeviceArray((0, 4), F32)).shape == (0, 16)


@pytest.mark.parametrize("slots,each,e", [(1, 1, 1), (63, 1, 5), (4096, 8, 3), (4100, 4, 3), (512 * 7, 2, 300), (40000, 8, 1024), (131072, 8, 128),
                                          (600000, 6, 61)])
def test_by_expert(slots, each, e):
    """stable, whole, and slots without an expert last"""
    g = rng(9, slots, e)
    which = g.integers(-1, e + 1, (slots // each, each)).astype(np.int32)
    which[g.random(which.shape) < 0.3] = e // 2
    which.reshape(-1)[::97] = np.iinfo(np.int32).min
    r = experts.by_expert(up(which), e)
    order, starts = oracle.by_expert(which, e)
    np.testing.assert_array_equal(r.starts.to_host(), starts)
    np.testing.assert_array_equal(r.order.to_host(), order)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("score,renorm", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
@pytest.mark.parametrize("rows,e,each", SIZES)
def test_route_backward(rows, e, each, score, renorm, kind):
    g = rng(10, rows, e, each)
    l = store(g.normal(0, 2, (rows, e)), kind)
    which = oracle.choose(wide(l), each, score)
    dw = g.normal(0, 1, (rows, each)).astype(F32)
    d = experts.route_backward(up(l), up(which), up(dw), score, renorm, 2.5)
    want, t = oracle.route_backward(wide(l), which, dw, score, renorm, 2.5)
    close(d.to_host(), want, 68 * 2.0 ** -24 * t, kind)


@pytest.mark.parametrize("score,renorm", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
def test_route_backward_by_differences(score, renorm):
    """the gradient of sum(dw * weights) against central differences of the definition's own weights (float64, a step of 1e-5:
    their error is 1e-10 of third derivatives below 10, and 1e-11 of rounding)"""
    g = rng(11)
    l = g.normal(0, 1, (6, 20)).astype(F32)
    which = oracle.choose(wide(l), 5, score)
    dw = g.normal(0, 1, (6, 5)).astype(F32)
    d = experts.route_backward(up(l), up(which), up(dw), score, renorm, 1.5).to_host()
    v = wide(l)
    for i in range(20):
        up_, down = v.copy(), v.copy()
        up_[:, i] += 1e-5
        down[:, i] -= 1e-5
        diff = ((oracle.weights(up_, which, score, renorm, 1.5) - oracle.weights(down, which, score, renorm, 1.5)) * dw).sum(1) / 2e-5
        np.testing.assert_allclose(d[:, i], diff, atol=68 * 2.0 ** -24 * 1.5 * 2 * abs(dw).sum(1).max() + 1e-8, rtol=0)


def test_route_backward_numbers_twice_and_outside():
    """an expert named twice gets both places' gradients, numbers outside are passed over, a row without any is zero"""
    g = rng(12)
    l = g.normal(0, 1, (5, 30)).astype(F32)
    l[3, 4:] = -np.inf
    which = np.array([[3, 3, 7], [-1, 2, 30], [-1, -5, 99], [0, 1, -1], [29, 29, 29]], np.int32)
    dw = g.normal(0, 1, (5, 3)).astype(F32)
    dw[2] = np.nan
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            want, t = oracle.route_backward(wide(l), which, dw, score, renorm, 1.0)
            close(experts.route_backward(up(l), up(which), up(dw), score, renorm).to_host(), want, 68 * 2.0 ** -24 * t, F32)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("e", [40, 200, 700])
def test_route_backward_of_masked_rows(e, renorm, score, kind):
    """a row whose logits are all -inf has no experts and a gradient of zeros, whatever dweights holds there; masked logits of
    other rows have zeros"""
    g = rng(19, e)
    l = g.normal(0, 1, (37, e))
    l[:, 1::3] = -np.inf
    l[::5] = -np.inf
    l = store(l, kind)
    r = experts.route(up(l), 8, score, renorm=renorm)
    which = r.which.to_host()
    assert (which[::5] == -1).all() and (r.weights.to_host()[::5] == 0).all()
    dw = g.normal(0, 1, (37, 8)).astype(F32)
    dw[::5] = np.nan
    got = wide(experts.route_backward(up(l), r.which, up(dw), score, renorm).to_host())
    assert (got[::5] == 0).all() and (got[:, 1::3] == 0).all()
    some = np.arange(37) % 5 > 0
    want, t = oracle.route_backward(wide(l[some]), which[some], dw[some], score, renorm, 1.0)
    close(store(got[some], kind), want, 68 * 2.0 ** -24 * t, kind)


@pytest.mark.parametrize("stride", [64, 67, 72])
def test_route_backward_strides(stride):
    g = rng(13)
    l, h = g.normal(0, 1, (9, 64)).astype(F32), np.full((9, stride), 5, F32)
    h[:, :64] = l
    base, to = up(h), up(np.full((9, stride), 3, F32))
    which, dw = oracle.choose(wide(l), 4, "softmax"), g.normal(0, 1, (9, 4)).astype(F32)
    view = lambda a: dev.DeviceArray((9, 64), F32, ptr=a.ptr, owner=a)
    experts.route_backward(view(base), up(which), up(dw), renorm=False, dlogits=view(to), logits_stride=stride, dlogits_stride=stride)
    got = to.to_host()
    want, t = oracle.route_backward(wide(l), which, dw, "softmax", False, 1.0)
    close(got[:, :64], want, 68 * 2.0 ** -24 * t, F32)
    assert (got[:, 64:] == 3).all()


JOINS = [(1, 1, 1), (1, 8, 4096), (3, 2, 7), (64, 4, 129), (33, 32, 8), (5, 3, 8200), (300, 6, 64)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,each,n", JOINS)
@pytest.mark.parametrize("masked", [False, True])
def test_join(rows, each, n, masked, kind):
    g = rng(14, rows, each, n)
    y, w = store(g.normal(0, 1, (rows * each, n)), kind), g.normal(0, 1, (rows, each)).astype(F32)
    which = None
    valid = np.ones((rows, each), bool)
    if masked:
        which = g.integers(-1, 5, (rows, each)).astype(np.int32)
        which[0] = -1                                # a row that has none
        valid = (which >= 0) & (which < 4)
        y[~valid.reshape(-1)] = store(np.array(np.nan), kind)
        w[~valid] = np.inf
    out = experts.join(up(y), up(w), None if which is None else up(which), 4 if masked else None)
    v, ww = np.where(valid.reshape(-1, 1), wide(y), 0).reshape(rows, each, n), np.where(valid, w, 0).astype(np.float64)[:, :, None]
    close(out.to_host(), (ww * v).sum(1), each * 2.0 ** -24 * abs(ww * v).sum(1), kind)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,each,n", JOINS)
@pytest.mark.parametrize("masked", [False, True])
def test_join_backward(rows, each, n, masked, kind):
    g = rng(15, rows, each, n)
    y, w = store(g.normal(0, 1, (rows * each, n)), kind), g.normal(0, 1, (rows, each)).astype(F32)
    d = store(g.normal(0, 1, (rows, n)), kind)
    which = g.integers(-1, 5, (rows, each)).astype(np.int32) if masked else None
    valid = np.ones((rows, each), bool) if which is None else (which >= 0) & (which < 4)
    if masked:
        y[~valid.reshape(-1)] = store(np.array(np.nan), kind)
    dy, dw = experts.join_backward(up(y), up(w), up(d), None if which is None else up(which), 4 if masked else None)
    dd = wide(d)[:, None]
    v, ww = np.where(valid.reshape(-1, 1), wide(y), 0).reshape(rows, each, n), np.where(valid, w, 0).astype(np.float64)[:, :, None]
    close(dy.to_host(), (ww * dd).reshape(rows * each, n), 2.0 ** -24 * abs(ww * dd).reshape(rows * each, n), kind)
    terms = np.where(valid[:, :, None], dd * v, 0)
    close(dw.to_host(), terms.sum(2), n * 2.0 ** -24 * abs(terms).sum(2), F32)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,stride,offset", [(64, 72, 0), (64, 67, 0), (61, 64, 0), (64, 64, 1)])
def test_join_strides(n, stride, offset, kind):
    """rows further apart, at addresses that no wide load takes; what lies between them stays"""
    g = rng(16, n, stride)
    rows, each = 13, 3
    hold = lambda m: store(g.normal(0, 1, m * stride + offset), kind)
    y, d, w = hold(rows * each), hold(rows), g.normal(0, 1, (rows, each)).astype(F32)
    size = np.dtype(kind).itemsize
    by, bd = up(y), up(d)
    bo, bdy = up(np.full(rows * stride + offset, 9, kind)), up(np.full(rows * each * stride + offset, 9, kind))
    view = lambda b, m: dev.DeviceArray((m, n), kind, ptr=b.ptr + offset * size, owner=b)
    cut = lambda a, m: a[offset:].reshape(m, stride)
    experts.join(view(by, rows * each), up(w), out=view(bo, rows), y_stride=stride, out_stride=stride)
    _, dw = experts.join_backward(view(by, rows * each), up(w), view(bd, rows), dy=view(bdy, rows * each), y_stride=stride, dout_stride=stride,
                                  dy_stride=stride)
    v, ww = wide(cut(y, rows * each)[:, :n]).reshape(rows, each, n), w.astype(np.float64)[:, :, None]
    got = cut(bo.to_host(), rows)
    close(got[:, :n], (ww * v).sum(1), each * 2.0 ** -24 * abs(ww * v).sum(1), kind)
    dd = wide(cut(d, rows)[:, :n])[:, None]
    gy = cut(bdy.to_host(), rows * each)
    close(gy[:, :n], (ww * dd).reshape(-1, n), 2.0 ** -24 * abs(ww * dd).reshape(-1, n), kind)
    close(dw.to_host(), (dd * v).sum(2), n * 2.0 ** -24 * abs(dd * v).sum(2), F32)
    nine = np.full(1, 9, kind)[0]
    assert (got[:, n:] == nine).all() and (gy[:, n:] == nine).all() and (bo.to_host()[:offset] == nine).all()


def last(a, rows):
    """the last rows of an array"""
    n = a.shape[1]
    return dev.DeviceArray((rows, n), a.dtype, ptr=a.ptr + (a.shape[0] - rows) * n * a.dtype.itemsize, owner=a)


def fill_last(a, h):
    check(lib().spa_memcpy_h2d(last(a, len(h)).ptr, h.ctypes.data, h.nbytes, None))


def test_logits_past_4_gib():
    rows, e, each = (1 << 32) // (256 * 2) + 70001, 256, 4
    g = rng(21)
    l = dev.DeviceArray((rows, e), BF16)
    l.zero()
    h = store(g.normal(0, 1, (50, e)), BF16)
    fill_last(l, h)
    r = experts.route(l, each, sort=False)
    want = oracle.choose(wide(h), each, "softmax")
    np.testing.assert_array_equal(last(r.which, 50).to_host(), want)
    close(last(r.weights, 50).to_host(), oracle.weights(wide(h), want, "softmax", True, 1.0), 2.0 ** -36, F32)
    dw = dev.DeviceArray((rows, each), F32)
    dw.zero()
    d = g.normal(0, 1, (50, each)).astype(F32)
    fill_last(dw, d)
    got = experts.route_backward(l, r.which, dw)
    want, t = oracle.route_backward(wide(h), want, d, "softmax", True, 1.0)
    close(last(got, 50).to_host(), want, 68 * 2.0 ** -24 * t, BF16)
    assert not dev.DeviceArray((1000, e), BF16, ptr=got.ptr, owner=got).to_host().any()


def test_joined_rows_past_4_gib():
    rows, each, n = 33001, 2, 33000
    g = rng(22)
    y, w, d = dev.DeviceArray((rows * each, n), BF16), dev.DeviceArray((rows, each), F32), dev.DeviceArray((rows, n), BF16)
    for a in (y, w, d):
        a.zero()
    hy, hw, hd = store(g.normal(0, 1, (6, n)), BF16), g.normal(0, 1, (3, each)).astype(F32), store(g.normal(0, 1, (3, n)), BF16)
    for a, h in ((y, hy), (w, hw), (d, hd)):
        fill_last(a, h)
    out = experts.join(y, w)
    terms = wide(hy).reshape(3, each, n) * wide(hw)[:, :, None]
    close(last(out, 3).to_host(), terms.sum(1), (each + 1) * 2.0 ** -24 * abs(terms).sum(1), BF16)
    dy, dw = experts.join_backward(y, w, d)
    close(last(dy, 6).to_host(), (wide(hd)[:, None] * wide(hw)[:, :, None]).reshape(6, n), 2.0 ** -24 * abs(wide(hd)[:, None] * wide(hw)[:, :, None]).reshape(6, n), BF16)
    dots = wide(hy).reshape(3, each, n) * wide(hd)[:, None]
    close(last(dw, 3).to_host(), dots.sum(2), n * 2.0 ** -24 * abs(dots).sum(2), F32)
    for a in (out, dy):
        assert not dev.DeviceArray((1000, n), BF16, ptr=a.ptr, owner=a).to_host().any()


def test_threads_at_once():
    """two threads, each with a stream of its own, route batches that need workspaces of different sizes"""
    found = []

    def work(seed, rows, e):
        st = dev.Stream()
        g = rng(17, seed)
        for _ in range(6):
            l = g.normal(0, 1, (rows, e)).astype(F32)
            x = dev.DeviceArray((rows, e), F32)
            check(lib().spa_memcpy_h2d(x.ptr, l.ctypes.data, l.nbytes, st.handle))
            r = experts.route(x, 6, stream=st.handle)
            st.synchronize()
            want = oracle.choose(wide(l), 6, "softmax")
            order, starts = oracle.by_expert(want, e)
            found.append(np.array_equal(r.which.to_host(stream=st.handle), want) and np.array_equal(r.order.to_host(stream=st.handle), order)
                         and np.array_equal(r.starts.to_host(stream=st.handle), starts))

    ts = [threading.Thread(target=work, args=a) for a in ((1, 3000, 96), (2, 5000, 200))]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert found == [True] * 12


def test_a_workspace_that_is_too_small_is_refused():
    x = up(rng(18).normal(0, 1, (5000, 64)).astype(F32))
    with pytest.raises(SpaError):
        experts.route(x, 4, work=dev.DeviceArray(256, np.uint8))


@pytest.mark.parametrize("e,groups", [(512, 8), (512, 64), (1024, 16), (290, 58), (64, 1)])
@pytest.mark.parametrize("rows", [1, 8])
def test_a_workspace_of_no_bytes_is_left_alone(rows, e, groups):
    """up to 8 rows need no workspace, in whichever form: a block that comes along with a length of 0, at any address, stays"""
    each = 3
    assert lib().spa_route_work_bytes(rows, e, each, 1) == 0
    l = rng(23, e, rows).normal(0, 1, (rows, e)).astype(F32)
    x, block = up(l), up(np.full(1 << 14, 0xa5, np.uint8))
    o = {"which": dev.DeviceArray((rows, each), np.int32), "weights": dev.DeviceArray((rows, each), F32), "order": dev.DeviceArray(rows * each, np.int32),
         "starts": dev.DeviceArray(e + 1, np.int32)}
    check(lib().spa_route(x.ptr, 2, rows, e, e, 0, None, groups, min(groups, 4), 2, each, 1, 1.0, *(a.ptr for a in o.values()), block.ptr + 1024, 0, None))
    want = oracle.choose(wide(l), each, "softmax", groups=groups, keep=min(groups, 4))
    order, starts = oracle.by_expert(want, e)
    for name, h in (("which", want), ("order", order), ("starts", starts)):
        np.testing.assert_array_equal(o[name].to_host(), h)
    assert (block.to_host() == 0xa5).all()


def test_join_backward_of_more_slots_than_one_launch_takes():
    """2^24 workgroups of 256 are one too many: the launches' ends lie inside a row"""
    each, n = 3, 2
    rows = (1 << 24) // each + 1001
    g = rng(24)
    turns = lambda a, m: np.ascontiguousarray(np.tile(a, (m // len(a) + 1, 1))[:m])
    y, w, d = turns(g.normal(0, 1, (997, n)).astype(F32), rows * each), turns(g.normal(0, 1, (991, each)).astype(F32), rows), turns(g.normal(0, 1, (983, n)).astype(F32), rows)
    dy, dw = experts.join_backward(up(y), up(w), up(d))
    dd = np.repeat(d, each, 0)
    np.testing.assert_array_equal(dy.to_host(), dd * w.reshape(-1, 1))         # one float32 product
    terms = dd.astype(np.float64) * y
    close(dw.to_host().reshape(-1), terms.sum(1), n * 2.0 ** -24 * abs(terms).sum(1), F32)


def test_keys_of_42_bits():
    """with a bias or groups, keys that agree to 42 bits of their mantissas are equal: the logistic of 31 and of 32 lies within 2^-43 of
    1, that of 29 does not"""
    l = np.full((2, 16), -1, F32)
    l[:, 9], l[0, 3], l[1, 3] = 32, 31, 29
    for one in (dict(bias=up(np.zeros(16, F32))), dict(groups=2, keep=2)):
        which = experts.route(up(l), 2, "sigmoid", **one).which.to_host()
        assert list(which[0]) == [3, 9] and list(which[1]) == [9, 3]
    assert (experts.route(up(l), 2, "sigmoid").which.to_host() == [9, 3]).all()       # the logits themselves are the keys
