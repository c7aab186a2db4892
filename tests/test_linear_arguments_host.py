"""Arguments that reach past their memory or mean something else than they say: errors before any device call."""
import numpy as np
import pytest

from seedpack_amd import device as dev
from seedpack_amd import linear
from seedpack_amd._lib import lib

P, ARG = 4096, -4


def memory(n, dtype=np.uint8):
    """n numbers of known extent, at no real address"""
    return dev.DeviceArray(n, dtype, ptr=1 << 20, owner=dev)


def part(of, shape, dtype, offset=0):
    return dev.DeviceArray(shape, dtype, ptr=of.ptr + offset, owner=of)


def own(shape, dtype):
    """an array as the library's allocations are, but for its address"""
    a = dev.DeviceArray(shape, dtype, ptr=1 << 20)
    a._owner = None
    a.__class__ = type("Own", (dev.DeviceArray,), {"__slots__": (), "__del__": lambda self: None})
    return a


def weight(rows=8, t=12, cols=256):
    return linear.Weight(t, memory(rows * 144 if t == 12 else 2 * rows * cols), rows, cols)


@pytest.mark.parametrize("call", [
    lambda x, out, far, of: linear.project(x, weight(), out=own((4, 8), np.uint16), out_stride=9),
    lambda x, out, far, of: linear.project(x, weight(), out=part(of, (4, 8), np.uint16), out_stride=of.nbytes // 6),
    lambda x, out, far, of: linear.project(far, weight(), out=out, x_stride=of.nbytes // 6),
    lambda x, out, far, of: linear.project(own((4, 256), np.uint16), weight(), out=out, x_stride=257),
    lambda x, out, far, of: linear.gated(far, weight(), weight(), out=out, x_stride=of.nbytes // 6),
    lambda x, out, far, of: linear.gated(x, weight(), weight(), out=own((4, 8), np.uint16), out_stride=16),
    lambda x, out, far, of: linear.gated_backward(x, weight(), weight(), own((4, 8), np.uint16), dx=part(of, (4, 256), np.uint16), dh_stride=10),
    lambda x, out, far, of: linear.gated_backward(x, weight(), weight(), out, dx=part(of, (4, 256), np.uint16), dx_stride=of.nbytes // 6),
    lambda x, out, far, of: linear.add_squares(far, part(of, (1, 256), np.float32), part(of, 1, np.int64), x_stride=of.nbytes // 6),
])
def test_strides_stay_within_their_memory(call):
    of = memory(1 << 16)
    x, out = part(of, (4, 256), np.uint16), part(of, (4, 8), np.uint16)
    with pytest.raises(ValueError, match="past its memory"):
        call(x, out, part(of, (4, 256), np.uint16), of)


def test_strides_that_fit():
    """the last row may end with the memory, one row has no stride, and a part's part counts for the whole"""
    of = memory(2 * (3 * 300 + 256))
    assert linear._rows("x", part(of, (4, 256), np.uint16), 300, 256) == (0, 4, 256, 300)
    assert linear._rows("x", part(part(of, 600, np.uint8), (4, 256), np.uint16), 300, 256) == (0, 4, 256, 300)
    assert linear._rows("x", own((1, 256), np.uint16), 1 << 40, 256) == (0, 1, 256, 1 << 40)
    assert linear._rows("x", own((0, 256), np.uint16), 300, 256) == (0, 0, 256, 300)
    assert linear._rows("x", memory((4, 256), np.uint16), 300, 256) == (0, 4, 256, 300)      # a framework's tensor behind it
    with pytest.raises(ValueError):
        linear._rows("x", part(of, (4, 256), np.uint16, 2), 300, 256)


def test_one_adapter_a_row():
    """numbers of adapters are one a row, not rows of them"""
    of = memory(1 << 16)
    x, out = part(of, (4, 256), np.uint16), part(of, (4, 8), np.uint16)
    pool = linear.Adapters(memory((2, 8, 256), np.uint16), memory((2, 8, 8), np.uint16), memory(2, np.float32))
    for shape in ((4, 2), (4, 4), (4, 1, 3)):
        with pytest.raises(ValueError):
            linear.project(x, weight(), pool, memory(shape, np.int32), out=out)


@pytest.mark.parametrize("each", [1 << 62, (1 << 62) + 1, (1 << 61) + 2, (1 << 63) - 1, 1 << 40])
def test_experts_of_a_row_beyond_counting(each):
    """numbers of experts whose product with the rows passes 64 bits"""
    assert lib().spa_add_squares(P, 0, 8, 64, 64, P, each, 3, P, P, P, 1 << 40, None) == ARG
