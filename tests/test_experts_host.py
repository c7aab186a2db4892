"""Arguments of the routing, the join and the 4-bit matrices that are refused, before any device call."""
import numpy as np
import pytest

from seedpack_amd import device as dev
from seedpack_amd import experts, mx4
from seedpack_amd._lib import lib

P, ARG, TYPE = 4096, -4, -2
U8, I32, F32 = np.uint8, np.int32, np.float32


def memory(shape, dtype):
    """an array at no real address"""
    return dev.DeviceArray(shape, dtype, ptr=1 << 20, owner=dev)


def matrix(rows, cols, count=1):
    return mx4.Matrix(memory((count * rows, 16 * mx4.pitch(cols)), U8), memory((count * rows, mx4.pitch(cols)), U8), rows, cols, count)


def test_pitch():
    for cols in (1, 32, 255, 256, 257, 4096, 4000000):
        assert mx4.pitch(cols) == lib().spa_mx4_pitch(cols) == -(-cols // 256) * 8
    assert lib().spa_mx4_pitch(0) == lib().spa_mx4_pitch(4000001) == 0


@pytest.mark.parametrize("change,code", [
    ({"kind": 3}, TYPE), ({"experts": 0}, ARG), ({"experts": 1025}, ARG), ({"stride": 15}, ARG), ({"score": 2}, ARG), ({"groups": 0}, ARG),
    ({"groups": 3}, ARG), ({"groups": 65, "experts": 130, "stride": 130}, ARG), ({"keep": 3}, ARG), ({"keep": 0}, ARG), ({"best": 3}, ARG),
    ({"each": 0}, ARG), ({"each": 33, "experts": 64, "stride": 64}, ARG), ({"each": 17}, ARG), ({"groups": 4, "keep": 1, "each": 5}, ARG),
    ({"order": None}, ARG), ({"logits": None}, ARG), ({"which": None}, ARG), ({"weights": None}, ARG), ({"rows": -1}, ARG), ({"rows": 1 << 31}, ARG),
    ({"rows": 1 << 30}, ARG), ({"rows": 5000, "work": None}, ARG), ({"rows": 5000, "work": P + 16}, ARG), ({"rows": 5000, "bytes": 255}, ARG)])
def test_route_refuses(change, code):
    a = dict(logits=P, kind=2, rows=8, experts=16, stride=16, score=0, bias=None, groups=2, keep=2, best=2, each=4, renorm=1, scale=1.0, which=P,
             weights=P, order=P, starts=P, work=P, bytes=1 << 20, stream=None) | change
    assert lib().spa_route(*a.values()) == code


@pytest.mark.parametrize("change,code", [({"kind": 5}, TYPE), ({"dstride": 15}, ARG), ({"each": 17}, ARG), ({"dlogits": None}, ARG), ({"which": None}, ARG),
                                         ({"dweights": None}, ARG), ({"score": -1}, ARG)])
def test_route_backward_refuses(change, code):
    a = dict(logits=P, kind=0, rows=8, experts=16, stride=16, score=0, each=4, renorm=1, scale=1.0, which=P, dweights=P, dlogits=P, dstride=16,
             stream=None) | change
    assert lib().spa_route_backward(*a.values()) == code


def test_by_expert_refuses():
    L = lib()
    for a in ((P, 8, 0, P, P, None, 0), (P, 8, 1025, P, P, None, 0), (P, -1, 4, P, P, None, 0), (None, 8, 4, P, P, None, 0), (P, 8, 4, None, P, None, 0),
              (P, 8, 4, P, None, None, 0), (P, 1 << 31, 4, P, P, None, 0), (P, 100000, 64, P, P, None, 0)):
        assert L.spa_by_expert(*a, None) == ARG
    assert L.spa_by_expert_work_bytes(64, 8) == 0 and L.spa_by_expert_work_bytes(100000, 64) > 0


@pytest.mark.parametrize("change,code", [({"kind": 3}, TYPE), ({"each": 0}, ARG), ({"n": 0}, ARG), ({"ldy": 63}, ARG), ({"ldo": 63}, ARG), ({"y": None}, ARG),
                                         ({"weights": None}, ARG), ({"out": None}, ARG), ({"experts": 0}, ARG), ({"rows": 1 << 30}, ARG)])
def test_join_refuses(change, code):
    a = dict(y=P, kind=0, rows=8, each=4, n=64, ldy=64, weights=P, which=P, experts=4, out=P, ldo=64, stream=None) | change
    assert lib().spa_join(*a.values()) == code
    b = dict(a, dout=P, ldd=64, dy=a["out"], ldq=a["ldo"], dweights=P)
    order = ("y", "kind", "rows", "each", "n", "ldy", "weights", "which", "experts", "dout", "ldd", "dy", "ldq", "dweights", "stream")
    assert lib().spa_join_backward(*[b[k] for k in order]) == code


def test_quantize_refuses():
    L = lib()
    good = dict(x=P, kind=0, rows=8, cols=64, stride=64, across=0, codes=P, scales=P, stream=None)
    for change, code in (({"kind": 3}, TYPE), ({"cols": 0}, ARG), ({"cols": 4000001, "stride": 4000001}, ARG), ({"stride": 63}, ARG), ({"x": None}, ARG),
                         ({"codes": None}, ARG), ({"codes": P + 8}, ARG), ({"scales": P + 4}, ARG), ({"rows": -1}, ARG), ({"across": 1, "rows": 0}, ARG),
                         ({"across": 1, "rows": 4000001}, ARG)):
        assert L.spa_mx4_quantize(*(good | change).values()) == code
    assert L.spa_mx4_values(P, P, 8, 64, P, 3, 64, None) == TYPE
    assert L.spa_mx4_values(P, P, 8, 64, P, 0, 63, None) == ARG
    assert L.spa_mx4_values(P, None, 8, 64, P, 0, 64, None) == ARG
    assert L.spa_mx4_from_blocks(P, 8, 48, P, P, None) == ARG
    assert L.spa_mx4_from_blocks(None, 8, 64, P, P, None) == ARG


@pytest.mark.parametrize("change,code", [
    ({"kind": 3}, TYPE), ({"k": 0}, ARG), ({"xc": None}, ARG), ({"ws": None}, ARG), ({"wc": P + 1}, ARG), ({"n": -1}, ARG), ({"ld": 63}, ARG), ({"y": None}, ARG),
    ({"experts": 1025}, ARG), ({"experts": -1}, ARG), ({"order": None}, ARG), ({"starts": None}, ARG), ({"slots": 20}, ARG),
    ({"xm": 0}, ARG), ({"xm": 1 << 25, "slots": 1 << 26}, ARG)])
def test_products_refuse(change, code):
    a = dict(xc=P, xs=P, xm=8, k=256, wc=P, ws=P, n=64, experts=4, order=P, starts=P, slots=16, y=P, kind=0, ld=64, work=P, bytes=1 << 40, stream=None) | change
    assert lib().spa_mx4_project(*a.values()) == code
    g = [a[k] for k in ("xc", "xs", "xm", "k", "wc", "ws")] + [P, P, a["n"], 0] + [a[k] for k in ("experts", "order", "starts", "slots", "y", "kind", "ld", "work", "bytes", "stream")]
    assert lib().spa_mx4_gated(*g) == code
    g[9] = 2
    assert lib().spa_mx4_gated(*g) == ARG
    g[6:8], g[9] = [None, P], 0
    assert lib().spa_mx4_gated(*g) in (code, ARG)


@pytest.mark.parametrize("call", [
    lambda: experts.Routing(memory((4, 2), np.int64)),
    lambda: experts.Routing(memory(8, I32)),
    lambda: experts.Routing(memory((4, 2), I32), memory(8, I32)),
    lambda: experts.Routing(memory((4, 2), I32), memory(7, I32), memory(5, I32)),
    lambda: experts.Routing(memory((4, 2), I32), weights=memory((2, 4), F32)),
    lambda: experts.route(memory((4, 8), F32), 2, score="max"),
    lambda: experts.route(memory((4, 8), F32), 2, bias=memory(7, F32)),
    lambda: experts.route(memory((4, 8), F32), 2, bias=memory(8, np.float64)),
    lambda: experts.route(memory((4, 8), np.float64), 2),
    lambda: experts.route(memory((4, 8), F32), 2, logits_stride=7),
    lambda: experts.route(memory((4, 8), F32), 2, which=memory((4, 3), I32)),
    lambda: experts.route(memory((4, 8), F32), 2, which=memory((4, 2), I32), weights=memory((4, 2), F32), order=memory(8, I32), starts=memory(8, I32)),
    lambda: experts.route(memory((4, 8), F32), 2, which=memory((4, 2), I32), weights=memory((4, 2), F32), order=memory(8, I32), sort=False),
    lambda: experts.route_backward(memory((4, 8), F32), memory((3, 2), I32), memory((3, 2), F32)),
    lambda: experts.route_backward(memory((4, 8), F32), memory((4, 2), I32), memory((4, 3), F32)),
    lambda: experts.route_backward(memory((4, 8), F32), memory((4, 2), I32), memory((4, 2), F32), dlogits=memory((4, 8), np.uint16)),
    lambda: experts.by_expert(memory(8, I32), 4),
    lambda: experts.join(memory((8, 16), F32), memory((3, 2), F32)),
    lambda: experts.join(memory((8, 16), F32), memory((4, 2), F32), which=memory((4, 2), I32)),
    lambda: experts.join(memory((8, 16), F32), memory((4, 2), F32), which=memory((8, 1), I32), experts=4),
    lambda: experts.join(memory((8, 16), F32), memory((4, 2), F32), out=memory((4, 16), np.uint16)),
    lambda: experts.join_backward(memory((8, 16), F32), memory((4, 2), F32), memory((8, 16), F32)),
    lambda: experts.join_backward(memory((8, 16), F32), memory((4, 2), F32), memory((4, 16), np.uint16)),
    lambda: mx4.Matrix(memory((4, 64), U8), memory((4, 8), U8), 4, 32),
    lambda: mx4.Matrix(memory((4, 128), np.int8), memory((4, 8), U8), 4, 32),
    lambda: mx4.Matrix(memory((4, 128), U8), memory((4, 8), U8), 4, 0),
    lambda: mx4.quantize(memory((4, 64), F32), out=matrix(4, 65)),
    lambda: mx4.quantize(memory((4, 64), F32), across=True, out=matrix(4, 64)),
    lambda: mx4.quantize(memory((4, 64), np.int8), out=matrix(4, 64)),
    lambda: mx4.values(matrix(4, 64), out=memory((4, 63), F32)),
    lambda: mx4.values(matrix(4, 64), out=memory((4, 64), np.int8)),
    lambda: mx4.from_blocks(memory(4 * 2 * 17 - 1, U8), 4, 64, out=matrix(4, 64)),
    lambda: mx4.from_blocks(memory(1 << 16, U8), 4, 48, out=matrix(4, 48)),
    lambda: mx4.from_blocks(memory(1 << 16, U8), 4, 64, out=matrix(4, 96)),
    lambda: mx4.project(matrix(4, 64), matrix(8, 96), out=memory((4, 8), F32)),
    lambda: mx4.project(matrix(4, 64), matrix(8, 64, 3), out=memory((12, 8), F32)),
    lambda: mx4.project(matrix(4, 64), matrix(8, 64, 3), experts.Routing(memory((4, 2), I32)), out=memory((8, 8), F32)),
    lambda: mx4.project(matrix(4, 64), matrix(8, 64, 3), experts.Routing(memory((4, 2), I32), memory(8, I32), memory(5, I32)), out=memory((8, 8), F32)),
    lambda: mx4.project(matrix(5, 64), matrix(8, 64, 3), experts.Routing(memory((4, 2), I32), memory(8, I32), memory(4, I32)), out=memory((8, 8), F32)),
    lambda: mx4.project(matrix(4, 64), matrix(8, 64), out=memory((4, 8), np.int8)),
    lambda: mx4.project(matrix(4, 64), matrix(8, 64), out=memory((4, 8), F32), out_stride=7),
    lambda: mx4.gated(matrix(4, 64), matrix(8, 64), matrix(9, 64), out=memory((4, 8), F32)),
    lambda: mx4.gated(matrix(4, 64), matrix(8, 64), matrix(8, 64), act="relu", out=memory((4, 8), F32)),
])
def test_python_refuses(call):
    with pytest.raises((ValueError, TypeError)):
        call()


def test_calls_past_one_launch_are_refused():
    """a dispatch counts its work-items in 32 bits; the sizes are the first that need 2^32"""
    L, w = lib(), (P, 1 << 60, None)
    for rows, e in ((1 << 28, 16), (1 << 27, 256), (1 << 28, 300)):
        assert L.spa_route(P, 0, rows, e, e, 0, None, 1, 1, 2, 1, 1, 1.0, P, P, None, None, None, 0, None) == ARG
        assert L.spa_route(P, 0, rows, e, e, 0, None, 1, 1, 2, 1, 1, 1.0, P, P, P, P, *w) == ARG
    assert L.spa_route(P, 0, 1 << 28, 16, 16, 0, None, 2, 1, 2, 1, 1, 1.0, P, P, P, P, *w) == ARG
    for rows, e in ((1 << 28, 16), (1 << 26, 300)):
        assert L.spa_route_backward(P, 0, rows, e, e, 0, 1, 1, 1.0, P, P, P, e, None) == ARG
    for kind, n in ((0, 64), (1, 57), (2, 32)):
        assert L.spa_join(P, kind, 1 << 29, 1, n, n, P, None, 0, P, n, None) == ARG
    assert L.spa_mx4_quantize(P, 0, 1 << 27, 256, 256, 0, P, P, None) == ARG
    assert L.spa_mx4_quantize(P, 0, 256, 1 << 29, 1 << 29, 1, P, P, None) == ARG
    assert L.spa_mx4_values(P, P, 1 << 30, 32, P, 0, 32, None) == ARG
    assert L.spa_mx4_from_blocks(P, 1 << 27, 256, P, P, None) == ARG
    m, n = 1 << 30, 3000
    assert L.spa_mx4_project(P, P, m, 256, P, P, n, 0, None, None, 0, P, 0, n, *w) == ARG
    assert L.spa_mx4_gated(P, P, m, 256, P, P, P, P, n, 0, 0, None, None, 0, P, 0, n, *w) == ARG


def test_few_rows_read_their_weights_once():
    """the form shows in the workspace: few rows of matrices past the cache are multiplied as they are read, in no pieces of k"""
    need = lib().spa_mx4_product_work_bytes
    assert need(1, 8192, 12288, 0, 0, 0) == need(4, 8192, 12288, 0, 0, 0) == 0
    assert need(1, 7168, 4096, 32, 4, 0) == need(1, 14336, 4096, 8, 2, 0) == need(1, 8192, 16384, 8, 1, 0) == 0
    assert need(32, 8192, 12288, 0, 0, 0) > 0 and need(32, 14336, 4096, 0, 0, 0) > 0          # too few tiles for the chip
