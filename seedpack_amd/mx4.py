"""4-bit floating point in microscaled blocks: 32 numbers of a sign, two bits of exponent and one of mantissa share a power of
two, and the matrix unit multiplies them as they lie.

  quantize     rows, or columns (for products that sum over rows: a weight's gradient), to a Matrix
  values       what a Matrix stands for
  from_blocks  a Matrix from a GGUF file's MXFP4 blocks
  project      products of two Matrices, x w^T; with a Routing each slot by its expert's matrix
  gated        the gated half of a feed-forward block of them, act(x gate^T) * (x up^T)

A Matrix of `count` matrices of `rows` rows of `cols` is codes (count * rows, 16 * pitch) uint8 and scales (count * rows,
pitch) uint8, pitch(cols) blocks a row. Products of codes and scales are exact, sums are float32, and each output is
rounded once. Arrays, streams, strides, workspaces and capture as in linear.

The reference has no counterpart: it codes the bytes of such tensors, and leaves their use to llama.cpp.
"""
import functools

import numpy as np

from . import device as dev
from ._lib import check, lib
from .linear import ACT, _KIND, _not_captured, _out, _rows, _scratch

_U8 = np.dtype(np.uint8)


def pitch(cols):
    """the blocks that a row of `cols` numbers takes: whole runs of eight"""
    return -(-cols // 256) * 8


@functools.lru_cache(256)
def _work_bytes(x_rows, cols, n, experts, slots, gated):
    return lib().spa_mx4_product_work_bytes(x_rows, cols, n, experts, slots, gated)


class Matrix:
    """`count` 4-bit matrices of `rows` rows of `cols` numbers, one behind another"""
    __slots__ = ("codes", "scales", "rows", "cols", "count")

    def __init__(self, codes, scales, rows, cols, count=1):
        if rows < 0 or cols <= 0 or count < 1:
            raise ValueError(f"bad shape {count} x {rows} x {cols}")
        need = count * rows * pitch(cols)
        if codes.dtype != _U8 or scales.dtype != _U8:
            raise TypeError(f"codes and scales are uint8, not {codes.dtype} and {scales.dtype}")
        if codes.nbytes < 16 * need or scales.nbytes < need:
            raise ValueError(f"{codes.nbytes} and {scales.nbytes} bytes hold no {count} x {rows} x {cols} codes and scales ({16 * need} and {need} bytes)")
        self.codes, self.scales, self.rows, self.cols, self.count = codes, scales, rows, cols, count


def empty(rows, cols, count=1, stream=None):
    """a Matrix of device memory that holds nothing yet"""
    _not_captured(stream, "result (out)")
    b = pitch(cols)
    return Matrix(dev.DeviceArray((count * rows, 16 * b), np.uint8), dev.DeviceArray((count * rows, b), np.uint8), rows, cols, count)


def _matrix(name, out, rows, cols, stream):
    if out is None:
        return empty(rows, cols, 1, stream)
    if (out.count * out.rows, out.cols) != (rows, cols):
        raise ValueError(f"{name} is {out.count} x {out.rows} x {out.cols}, {rows} x {cols} is needed")
    return out


def quantize(x, across=False, out=None, x_stride=None, stream=None):
    """x (rows, cols) -> Matrix of its rows, or, across, of its columns (cols rows of `rows` numbers)"""
    kind, m, k, ld = _rows("x", x, x_stride)
    out = _matrix("out", out, *((k, m) if across else (m, k)), stream)
    check(lib().spa_mx4_quantize(x.ptr, kind, m, k, ld, bool(across), out.codes.ptr, out.scales.ptr, stream))
    return out


def values(q, out=None, dtype=np.float32, out_stride=None, stream=None):
    """the numbers that a Matrix stands for, (count * rows, cols), of out's type or dtype (bf16 bits as uint16)"""
    m = q.count * q.rows
    out, ld = _out("out", out, m, q.cols, dtype if out is None else out.dtype, out_stride, stream)
    if out.dtype not in _KIND:
        raise TypeError(f"out must be bf16 bits (uint16), float16 or float32, not {out.dtype}")
    check(lib().spa_mx4_values(q.codes.ptr, q.scales.ptr, m, q.cols, out.ptr, _KIND[out.dtype], ld, stream))
    return out


def from_blocks(blocks, rows, cols, count=1, out=None, stream=None):
    """count matrices of GGUF MXFP4 blocks, 17 bytes for 32 numbers, as they lie in a file -> Matrix: the bytes of a gguf.Tensor
    of type gguf.MXFP4, whose shape is (cols, rows) or (cols, rows, count)"""
    if cols % 32:
        raise ValueError(f"rows of {cols} are not whole blocks of 32")
    need = count * rows * (cols // 32) * 17
    if blocks.nbytes < need:
        raise ValueError(f"{blocks.nbytes} bytes hold no {count} x {rows} x {cols} numbers ({need} bytes)")
    if out is None:
        out = empty(rows, cols, count, stream)
    elif (out.count, out.rows, out.cols) != (count, rows, cols):
        raise ValueError(f"out is {out.count} x {out.rows} x {out.cols}, {count} x {rows} x {cols} is needed")
    check(lib().spa_mx4_from_blocks(blocks.ptr, count * rows, cols, out.codes.ptr, out.scales.ptr, stream))
    return out


def _product(x, w, routing, out, dtype, out_stride, stream):
    """-> (out, its stride, kind, experts, order, starts, slots)"""
    if x.cols != w.cols or x.count != 1:
        raise ValueError(f"x is {x.count} x {x.rows} x {x.cols} beside weights of {w.cols} columns")
    if routing is None:
        if w.count != 1:
            raise ValueError(f"{w.count} matrices need a routing")
        slots, experts, order, starts = x.rows, 0, None, None
    else:
        if routing.order is None or routing.experts != w.count:
            raise ValueError("a routing without its order" if routing.order is None else f"a routing over {routing.experts} experts for {w.count} matrices")
        slots, experts, order, starts = routing.which.size, w.count, routing.order.ptr, routing.starts.ptr
        if x.rows not in (routing.which.shape[0], slots):
            raise ValueError(f"{x.rows} rows for a routing of {routing.which.shape[0]} rows and {slots} slots")
    out, ld = _out("out", out, slots, w.rows, np.dtype(dtype) if out is None else out.dtype, out_stride, stream)
    if out.dtype not in _KIND:
        raise TypeError(f"out must be bf16 bits (uint16), float16 or float32, not {out.dtype}")
    return out, ld, _KIND[out.dtype], experts, order, starts, slots


def project(x, w, routing=None, out=None, dtype=np.uint16, out_stride=None, work=None, stream=None):
    """x (rows of w.cols) -> (rows, w.rows): x w^T. With a routing of w.count experts, (slots, w.rows): slot p by its expert's
    matrix, from row p of x, or from row p // each where x has a row for each of the routing's; rows of slots without an
    expert are left as they are. Of out's type or dtype (bf16 bits as uint16)."""
    out, ld, kind, experts, order, starts, slots = _product(x, w, routing, out, dtype, out_stride, stream)
    keep, p, n = _scratch(_work_bytes(x.rows, x.cols, w.rows, experts, slots, 0), work, stream)
    check(lib().spa_mx4_project(x.codes.ptr, x.scales.ptr, x.rows, x.cols, w.codes.ptr, w.scales.ptr, w.rows, experts, order, starts, slots,
                            out.ptr, kind, ld, p, n, stream))
    return out


def gated(x, gate, up, act="silu", routing=None, out=None, dtype=np.uint16, out_stride=None, work=None, stream=None):
    """act(x gate^T) * (x up^T), act "silu" or "gelu" (tanh form); rows, slots and types as project"""
    if (gate.rows, gate.cols, gate.count) != (up.rows, up.cols, up.count):
        raise ValueError(f"gate is {gate.count} x {gate.rows} x {gate.cols}, up {up.count} x {up.rows} x {up.cols}")
    if act not in ACT:
        raise ValueError(f"unknown activation {act!r}: {sorted(ACT)}")
    out, ld, kind, experts, order, starts, slots = _product(x, gate, routing, out, dtype, out_stride, stream)
    keep, p, n = _scratch(_work_bytes(x.rows, x.cols, gate.rows, experts, slots, 1), work, stream)
    check(lib().spa_mx4_gated(x.codes.ptr, x.scales.ptr, x.rows, x.cols, gate.codes.ptr, gate.scales.ptr, up.codes.ptr, up.scales.ptr,
                          gate.rows, ACT[act], experts, order, starts, slots, out.ptr, kind, ld, p, n, stream))
    return out
