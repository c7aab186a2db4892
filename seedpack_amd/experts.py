"""A mixture of experts around the products with packed weights: which of a model's experts each row goes to, and what
their results come to.

  route           each row's experts and their weights, from the logits of a router; route_backward: the logits' gradient
  by_expert       the rows' slots in the order of their experts, for products by expert (mx4.project, mx4.gated)
  join            the weighted sum of each row's results; join_backward: its gradients

A slot is a row's place for one expert: row * each + j. `which`, (rows, each) int32, is what linear.add_squares takes too;
a number outside 0..experts-1 is a slot without an expert. Logits and results are DeviceArrays of BF16 bits (uint16), float16
or float32, row-major, with a `*_stride` (in elements) as in linear; which, weights, order and starts are dense. Every call
only queues work on `stream`; workspaces and results are kept and made as linear's are, and a captured call is given
both.

The reference has no counterpart: it packs a mixture's tensors like any others and leaves their use to llama.cpp.
"""
import functools

import numpy as np

from . import device as dev
from ._lib import check, lib
from .linear import _ids, _not_captured, _out, _rows, _scratch

SCORE = {"softmax": 0, "sigmoid": 1}
_I32, _F32 = np.dtype(np.int32), np.dtype(np.float32)


@functools.lru_cache(256)
def _route_work_bytes(rows, experts, each):
    return lib().spa_route_work_bytes(rows, experts, each, 1)


class Routing:
    """which (rows, each) int32, the slots' order (rows * each,) int32 and starts (experts + 1,) int32 (None both where not
    asked for), and weights (rows, each) float32 or None"""
    __slots__ = ("which", "order", "starts", "weights")

    def __init__(self, which, order=None, starts=None, weights=None):
        if which.dtype != _I32 or len(which.shape) != 2:
            raise ValueError(f"which is {which.shape} {which.dtype}: (rows, each) int32 is taken")
        if (order is None) != (starts is None):
            raise ValueError("order and starts go together")
        if order is not None and (order.dtype != _I32 or starts.dtype != _I32 or order.size != which.size or starts.size < 2):
            raise ValueError(f"order {order.shape} {order.dtype} and starts {starts.shape} {starts.dtype} for {which.size} slots")
        if weights is not None and (weights.dtype != _F32 or weights.shape != which.shape):
            raise ValueError(f"weights {weights.shape} {weights.dtype} beside which {which.shape}")
        self.which, self.order, self.starts, self.weights = which, order, starts, weights

    @classmethod
    def _of(cls, which, order, starts, weights):
        """of arrays that a call here has looked at"""
        r = cls.__new__(cls)
        r.which, r.order, r.starts, r.weights = which, order, starts, weights
        return r

    @property
    def experts(self):
        return self.starts.size - 1


def _made(name, a, shape, dtype, stream):
    if a is None:
        _not_captured(stream, f"result ({name})")
        return dev.DeviceArray(shape, dtype)
    if a.dtype is not dtype and a.dtype != dtype or a.shape != shape:
        raise ValueError(f"{name} is {a.shape} {a.dtype}, {shape} {dtype} is needed")
    return a


def _score(score):
    if score not in SCORE:
        raise ValueError(f"unknown score {score!r}: {sorted(SCORE)}")
    return SCORE[score]


def route(logits, each, score="softmax", bias=None, groups=1, keep=1, best=2, renorm=True, scale=1.0, sort=True, which=None,
          weights=None, order=None, starts=None, logits_stride=None, work=None, stream=None):
    """logits (rows, experts) -> Routing: each row's `each` experts of the largest keys, the best first (of equal ones the
    lowest number). score "softmax" (over the row) or "sigmoid"; keys are the logits, or, with a bias (experts,) float32 or
    groups, score + bias. groups: the experts are that many equal runs, of which the `keep` best take part; a run is worth
    the sum of its `best` (1 or 2) highest keys. (score + bias is a sum in 64 bits; sums that agree to 42 bits of their mantissas are
    equal, as the logistics of all logits above 30 are.) A logit of -inf is never chosen; a row with too few experts has -1
    and weight 0 in its last places. Weights are scale * score, with renorm divided by the sum of the row's chosen scores. sort:
    the slots' order too."""
    kind, m, e, ld = _rows("logits", logits, logits_stride)
    score = _score(score)
    if bias is not None and (bias.dtype != _F32 or bias.size != e):
        raise ValueError(f"bias {bias.shape} {bias.dtype} for {e} experts (float32)")
    which = _made("which", which, (m, each), _I32, stream)
    weights = _made("weights", weights, (m, each), _F32, stream)
    L = lib()
    p, n = None, 0
    if sort:
        order = _made("order", order, (m * each,), _I32, stream)
        starts = _made("starts", starts, (e + 1,), _I32, stream)
        held, p, n = _scratch(_route_work_bytes(m, e, each), work, stream)
    elif order is not None or starts is not None:
        raise ValueError("order and starts are written with sort only")
    check(L.spa_route(logits.ptr, kind, m, e, ld, score, None if bias is None else bias.ptr, groups, keep, best, each, bool(renorm),
                      scale, which.ptr, weights.ptr, order.ptr if sort else None, starts.ptr if sort else None, p, n, stream))
    return Routing._of(which, order, starts, weights)


def route_backward(logits, which, dweights, score="softmax", renorm=True, scale=1.0, dlogits=None, logits_stride=None,
                   dlogits_stride=None, stream=None):
    """the gradient of route()'s logits from its weights' (rows, each) float32: (rows, experts) of the logits' type, every
    number written. The choice itself and the bias have none."""
    kind, m, e, ld = _rows("logits", logits, logits_stride)
    score = _score(score)
    _ids(which, m)
    if len(which.shape) != 2 or dweights.dtype != _F32 or dweights.shape != which.shape:
        raise ValueError(f"dweights {dweights.shape} {dweights.dtype} beside which {which.shape}")
    dlogits, ldd = _out("dlogits", dlogits, m, e, logits.dtype, dlogits_stride, stream)
    check(lib().spa_route_backward(logits.ptr, kind, m, e, ld, score, which.shape[1], bool(renorm), scale, which.ptr, dweights.ptr,
                                   dlogits.ptr, ldd, stream))
    return dlogits


def by_expert(which, experts, order=None, starts=None, work=None, stream=None):
    """which (rows, each) int32 -> Routing with the slots in the order of their experts (those of one expert in their own, those
    without an expert last) and where each expert's begin"""
    if which.dtype != _I32 or len(which.shape) != 2:
        raise ValueError(f"which is {which.shape} {which.dtype}: (rows, each) int32 is taken")
    order = _made("order", order, (which.size,), _I32, stream)
    starts = _made("starts", starts, (experts + 1,), _I32, stream)
    L = lib()
    keep, p, n = _scratch(L.spa_by_expert_work_bytes(which.size, experts), work, stream)
    check(L.spa_by_expert(which.ptr, which.size, experts, order.ptr, starts.ptr, p, n, stream))
    return Routing._of(which, order, starts, None)


def _slots(y, weights, which, experts, y_stride):
    kind, slots, n, ld = _rows("y", y, y_stride)
    if weights.dtype != _F32 or len(weights.shape) != 2 or weights.size != slots or not weights.shape[1]:
        raise ValueError(f"weights {weights.shape} {weights.dtype} for {slots} rows of results: (rows, each) float32 is taken")
    if (which is None) != (experts is None):
        raise ValueError("which and the number of experts go together")
    if which is not None and (which.dtype != _I32 or which.shape != weights.shape):
        raise ValueError(f"which {which.shape} {which.dtype} beside weights {weights.shape}")
    return kind, weights.shape[0], weights.shape[1], n, ld


def join(y, weights, which=None, experts=None, out=None, y_stride=None, out_stride=None, stream=None):
    """y (rows * each, n), weights (rows, each) float32 -> (rows, n): the weighted sum of each row's results. With which and the
    number of experts, slots without an expert are passed over, whatever y and weights hold there."""
    kind, m, each, n, ld = _slots(y, weights, which, experts, y_stride)
    out, ldo = _out("out", out, m, n, y.dtype, out_stride, stream)
    check(lib().spa_join(y.ptr, kind, m, each, n, ld, weights.ptr, None if which is None else which.ptr, experts or 0, out.ptr, ldo,
                         stream))
    return out


def join_backward(y, weights, dout, which=None, experts=None, dy=None, dweights=None, y_stride=None, dout_stride=None, dy_stride=None,
                  stream=None):
    """the gradients of join() from dout (rows, n) -> dy (rows * each, n) of y's type, dweights (rows, each) float32; zeros for
    slots without an expert"""
    kind, m, each, n, ld = _slots(y, weights, which, experts, y_stride)
    _, mo, _, ldd = _rows("dout", dout, dout_stride, n)
    if mo != m or dout.dtype != y.dtype:
        raise ValueError(f"dout is {dout.shape} {dout.dtype} for {m} rows of {y.dtype}")
    dy, ldy = _out("dy", dy, m * each, n, y.dtype, dy_stride, stream)
    dweights = _made("dweights", dweights, (m, each), _F32, stream)
    check(lib().spa_join_backward(y.ptr, kind, m, each, n, ld, weights.ptr, None if which is None else which.ptr, experts or 0, dout.ptr,
                                  ldd, dy.ptr, ldy, dweights.ptr, stream))
    return dy, dweights
