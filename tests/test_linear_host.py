"""Refusals of the products with packed weights: every bad argument is an error before any device call."""
import numpy as np
import pytest

from seedpack_amd import device as dev
from seedpack_amd import linear
from seedpack_amd._lib import lib

P = 4096                                     # a pointer that no refused call reads


def project(type=12, w=P, n=8, k=256, kind=0, x=P, m=4, xs=256, y=P, ys=8, a=None, b=None, scale=None, pool=0, rank=0,
            which=None, work=P, work_bytes=1 << 40):
    return lib().spa_project(type, w, n, k, kind, x, m, xs, y, ys, a, b, scale, pool, rank, which, work, work_bytes, None)


def gated(type=12, gate=P, up=P, n=8, k=256, kind=0, x=P, m=4, xs=256, act=0, h=P, hs=8, work=P, work_bytes=1 << 40):
    return lib().spa_gated(type, gate, up, n, k, kind, x, m, xs, act, h, hs, work, work_bytes, None)


def backward(type=30, gate=P, up=P, n=8, k=256, kind=0, x=P, m=4, xs=256, act=0, dh=P, dhs=8, dx=P, dxs=256, dgate=P, dup=P,
             work=P, work_bytes=1 << 40):
    return lib().spa_gated_backward(type, gate, up, n, k, kind, x, m, xs, act, dh, dhs, dx, dxs, dgate, dup, work, work_bytes, None)


def squares(x=P, kind=0, rows=200, cols=64, xs=64, which=None, each=0, experts=0, sums=P, counts=P, work=P, work_bytes=1 << 40):
    return lib().spa_add_squares(x, kind, rows, cols, xs, which, each, experts, sums, counts, work, work_bytes, None)


TYPE, ARG = -2, -4
ADAPTERS = dict(a=P, b=P, scale=P, pool=2, rank=8, which=P)


@pytest.mark.parametrize("want,args", [
    (TYPE, dict(type=99)), (TYPE, dict(type=0)), (TYPE, dict(kind=2)), (TYPE, dict(kind=-1)),
    (ARG, dict(k=100)), (ARG, dict(k=0)), (ARG, dict(n=-1)), (ARG, dict(m=-1)), (ARG, dict(xs=255)), (ARG, dict(ys=7)),
    (ARG, dict(w=None)), (ARG, dict(x=None)), (ARG, dict(y=None)), (ARG, dict(x=P + 1)), (ARG, dict(y=P + 1)),
    (ARG, dict(type=30, w=P + 8)), (ARG, dict(k=1 << 23, xs=1 << 23)),
    (ARG, dict(pool=-1)), (ARG, dict(ADAPTERS, rank=0)), (ARG, dict(ADAPTERS, rank=257)), (ARG, dict(ADAPTERS, a=None)),
    (ARG, dict(ADAPTERS, b=None)), (ARG, dict(ADAPTERS, scale=None)), (ARG, dict(ADAPTERS, which=None)),
    (ARG, dict(ADAPTERS, a=P + 1)), (ARG, dict(ADAPTERS, which=P + 2)),
    (ARG, dict(work=None)), (ARG, dict(work=P + 16)), (ARG, dict(work_bytes=16)), (ARG, dict(m=1 << 31)),
])
def test_project(want, args):
    assert project(**args) == want
    assert b"spa_project" in lib().spa_last_error()


@pytest.mark.parametrize("want,args", [
    (TYPE, dict(type=99)), (TYPE, dict(kind=2)), (ARG, dict(act=2)), (ARG, dict(act=-1)), (ARG, dict(k=100)), (ARG, dict(hs=7)),
    (ARG, dict(xs=1)), (ARG, dict(gate=None)), (ARG, dict(up=None)), (ARG, dict(h=None)), (ARG, dict(h=P + 1)),
    (ARG, dict(type=1, kind=1, up=P + 2)), (ARG, dict(work_bytes=0)),
])
def test_gated(want, args):
    assert gated(**args) == want
    assert b"spa_gated" in lib().spa_last_error()


@pytest.mark.parametrize("want,args", [
    (TYPE, dict(type=99)), (TYPE, dict(type=12)), (TYPE, dict(type=1)), (ARG, dict(dgate=None)), (ARG, dict(dup=None)),
    (ARG, dict(act=7)), (ARG, dict(dhs=7)), (ARG, dict(dxs=255)), (ARG, dict(dh=None)), (ARG, dict(x=None)), (ARG, dict(dx=P + 1)),
    (ARG, dict(dgate=P + 1)), (ARG, dict(work=None)), (ARG, dict(work_bytes=1024)), (ARG, dict(n=1 << 22, dhs=1 << 22)),
])
def test_gated_backward(want, args):
    assert backward(**args) == want
    assert b"spa_gated_backward" in lib().spa_last_error()


@pytest.mark.parametrize("want,args", [
    (TYPE, dict(kind=3)), (ARG, dict(rows=-1)), (ARG, dict(cols=0)), (ARG, dict(xs=63)), (ARG, dict(experts=3)),
    (ARG, dict(which=P, experts=0, each=1)), (ARG, dict(which=P, experts=3, each=0)), (ARG, dict(which=P, experts=1 << 17, each=1)),
    (ARG, dict(x=None)), (ARG, dict(sums=None)), (ARG, dict(counts=None)), (ARG, dict(x=P + 1)), (ARG, dict(kind=2, x=P + 2)),
    (ARG, dict(sums=P + 2)), (ARG, dict(counts=P + 4)), (ARG, dict(work=None)), (ARG, dict(work_bytes=3)), (ARG, dict(work=P + 8)),
    (ARG, dict(which=P, experts=3, each=1 << 25)),
])
def test_add_squares(want, args):
    assert squares(**args) == want
    assert b"spa_add_squares" in lib().spa_last_error()


def test_nothing_to_do():
    assert project(m=0, x=None, y=None, work=None) == 0
    assert project(n=0, w=None, y=None, ys=0, work=None) == 0
    assert gated(m=0, x=None, h=None, work=None) == 0
    assert backward(m=0, dgate=None, dup=None, work=None) == 0
    assert backward(dx=None, dgate=None, dup=None, work=None) == 0
    assert squares(rows=0, x=None, work=None) == 0


def test_work_sizes():
    L = lib()
    assert L.spa_project_work_bytes(12, 8, 100, 0, 4, 0, 0) == 0 and L.spa_gated_work_bytes(99, 8, 256, 0, 4) == 0
    for t in (1, 30, 2, 8, 12, 18, 42):
        for m in (1, 3, 64, 65, 129, 300, 2053):
            plain = L.spa_project_work_bytes(t, 1000, 2048, 0, m, 0, 0)
            assert plain % 256 == 0 and L.spa_project_work_bytes(t, 1000, 2048, 0, m, 4, 16) > plain >= 2 * 2048 * m
            # weights of the inputs' type are multiplied as they lie, others are there once more as binary16 (twice beside F16)
            if m > 128 and t != 30:
                assert plain >= 2 * 1000 * 2048
            assert L.spa_gated_backward_work_bytes(t, 1000, 2048, 0, m, 1, 0) > L.spa_gated_backward_work_bytes(t, 1000, 2048, 0, m, 0, 0)
    assert L.spa_add_squares_work_bytes(5, 64, 0) == 0 and L.spa_add_squares_work_bytes(5000, 64, 0) > 0


def array(shape, dtype):
    return dev.DeviceArray(shape, dtype, ptr=P, owner=dev)


def test_python_refusals():
    x, w = array((4, 256), np.uint16), linear.Weight(12, array(8 * 144, np.uint8), 8, 256)
    bad = [
        lambda: linear.Weight(12, array(8 * 144, np.uint8), 8, 255),                         # not whole blocks
        lambda: linear.Weight(12, array(8 * 144 - 1, np.uint8), 8, 256),                     # too few bytes
        lambda: linear.Weight(5, array(4096, np.uint8), 8, 256),                             # no such type
        lambda: linear.project(array((4, 255), np.uint16), w),                               # columns
        lambda: linear.project(array((1024,), np.uint16), w),                                # not a matrix
        lambda: linear.project(array((4, 256), np.uint8), w),                                # type of the inputs
        lambda: linear.project(x, w, x_stride=255),
        lambda: linear.project(x, w, out=array((4, 9), np.uint16)),
        lambda: linear.project(x, w, out=array((4, 8), np.float16)),
        lambda: linear.project(x, w, out_stride=9),                                          # a stride of nothing
        lambda: linear.Adapters(array((2, 8, 256), np.uint16), array((2, 8, 4), np.uint16), array(2, np.float32)),
        lambda: linear.Adapters(array((2, 8, 256), np.uint16), array((2, 8, 8), np.float16), array(2, np.float32)),
        lambda: linear.Adapters(array((2, 8, 256), np.uint16), array((2, 8, 8), np.uint16), array(3, np.float32)),
        lambda: linear.gated(x, w, linear.Weight(12, array(9 * 144, np.uint8), 9, 256)),     # two shapes
        lambda: linear.gated(x, w, w, act="relu"),
        lambda: linear.gated_backward(x, w, w, array((4, 7), np.uint16)),
        lambda: linear.gated_backward(x, w, w, array((4, 8), np.float16)),
        lambda: linear.gated_backward(x, w, w, array((4, 8), np.uint16), dgate=array((8, 256), np.uint16)),
        lambda: linear.add_squares(x, array((1, 255), np.float32), array((1,), np.int64)),
        lambda: linear.add_squares(x, array((1, 256), np.float64), array((1,), np.int64)),
        lambda: linear.add_squares(x, array((2, 256), np.float32), array((2,), np.int64)),   # experts without numbers
        lambda: linear.add_squares(x, array((2, 256), np.float32), array((2,), np.int64), array((3, 1), np.int32)),
        lambda: linear.add_squares(x, array((2, 256), np.float32), array((2,), np.int64), array((4, 1), np.int64)),
    ]
    ad = linear.Adapters(array((2, 8, 256), np.uint16), array((2, 8, 8), np.uint16), array(2, np.float32))
    bad += [lambda: linear.project(x, w, ad), lambda: linear.project(x, w, ad, array((3,), np.int32)),
            lambda: linear.project(x, w, ad, array((4,), np.int64)),
            lambda: linear.project(array((4, 256), np.float16), w, ad, array((4,), np.int32))]
    for i, f in enumerate(bad):
        with pytest.raises((ValueError, TypeError)):
            f()
            pytest.fail(f"refusal {i} was taken")


def test_sizes_beyond_the_limits():
    """sizes are answered at once, whatever is asked"""
    L = lib()
    assert L.spa_add_squares_work_bytes(1000, 200000, 65535) == 0                  # one run: nothing to join
    assert L.spa_add_squares_work_bytes(5000, 200000, 65535) == 0
    assert L.spa_add_squares_work_bytes(1000, 4096, 1 << 20) == 0
    assert L.spa_project_work_bytes(12, 64, 256, 0, 300, 1 << 40, 1 << 40) == 0
    assert squares(which=P, rows=1000, cols=1 << 30, xs=1 << 30, experts=65535, each=1) == ARG
