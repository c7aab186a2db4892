"""Products with packed weights: what a program does with the tensors that this package regrows.

  project         a shared projection beside the low-rank adapters of the requests in a batch
  gated           the gated half of a feed-forward block, act(x gate^T) * (x up^T)
  gated_backward  its gradients
  add_squares     the column sums of squares that an importance matrix is made of

Weights are BF16 or F16 matrices or any of the 20 GGUF block types, as they lie in a file (`Weight`).
Inputs and outputs are two-dimensional DeviceArrays of BF16 bits (uint16) or float16, row-major; with a
`*_stride` (in elements) an array's rows may lie further apart than their columns: the array is then a part of
another one (`DeviceArray(shape, dtype, ptr=.., owner=other)`), which its last row has to end in. Every call only
queues work on `stream` and returns; results are float32 sums rounded once. A call's scratch is the calling
thread's own for that device and stream, kept between calls (until the stream ends or `release`), or is given as
`work`. Arrays that a call makes for its results come from the thread's cache of device blocks, whose work is on
one stream (device._Cache): a thread that uses several gives its own. A call that is captured into a graph is
given both, with workspaces of the C entries' `*_work_bytes`.

The reference has no counterpart: it makes and packs weights (seedpack/gpuquant.py:284-456) and leaves
their use to llama.cpp.
"""
import ctypes
import threading
import weakref

import numpy as np

from . import device as dev
from ._lib import check, lib
from .requant import QFUN

F16, BF16 = 1, 30
ACT = {"silu": 0, "gelu": 1}
_KIND = {np.dtype(np.uint16): 0, np.dtype(np.float16): 1, np.dtype(np.float32): 2}


class Weight:
    """a matrix of `rows` output rows of `cols` inputs: ggml type (F16, BF16 or a block type) and its bytes"""
    __slots__ = ("type", "data", "rows", "cols")

    def __init__(self, ttype, data, rows, cols):
        if ttype in (F16, BF16):
            need = 2 * rows * cols
        elif ttype in QFUN:
            _, qk, bs = QFUN[ttype]
            if cols % qk:
                raise ValueError(f"rows of {cols} weights are not whole blocks of {qk} (type {ttype})")
            need = rows * (cols // qk) * bs
        else:
            raise ValueError(f"unknown ggml type {ttype}")
        if rows < 0 or cols <= 0:
            raise ValueError(f"bad shape {rows} x {cols}")
        if data.nbytes < need:
            raise ValueError(f"{data.nbytes} bytes hold no {rows} x {cols} weights of type {ttype} ({need} bytes)")
        self.type, self.data, self.rows, self.cols = ttype, data, rows, cols


class Adapters:
    """a pool of low-rank adapters of one projection: a (count, rank, cols), b (count, rows, rank), both of the
    inputs' type, scale (count,) float32; number i adds scale[i] x a[i]^T b[i]^T"""
    __slots__ = ("a", "b", "scale", "count", "rank")

    def __init__(self, a, b, scale):
        if len(a.shape) != 3 or len(b.shape) != 3 or a.shape[0] != b.shape[0] or a.shape[1] != b.shape[2]:
            raise ValueError(f"adapters of shapes {a.shape} and {b.shape}: (count, rank, cols) and (count, rows, rank) are taken")
        self.count, self.rank = a.shape[:2]
        if scale.dtype != np.float32 or scale.size != self.count:
            raise ValueError(f"{scale.size} scales of {scale.dtype} for {self.count} adapters (float32)")
        if a.dtype != b.dtype:
            raise TypeError(f"adapters of two types, {a.dtype} and {b.dtype}")
        self.a, self.b, self.scale = a, b, scale


def _within(name, a, m, n, stride):
    """rows further apart than an array's columns lie inside the array that it is a part of; memory that is not a
    DeviceArray's own (a framework's tensor behind it) is the caller's word"""
    if m and stride != n:
        last, of = a.ptr + ((m - 1) * stride + n) * a.dtype.itemsize, a
        while isinstance(of._owner, dev.DeviceArray) and of._owner is not of:
            of = of._owner
        if (of is not a or of._owner is None) and last > of.ptr + of.nbytes:
            raise ValueError(f"{name}: {m} rows of {n} at a stride of {stride} reach {last - of.ptr - of.nbytes} bytes past its memory")


def _rows(name, a, stride, cols=None):
    """a 2-D array -> (kind, rows, columns, stride)"""
    kind = _KIND.get(a.dtype)
    if kind is None:
        raise TypeError(f"{name} must be bf16 bits (uint16), float16 or float32, not {a.dtype}")
    if len(a.shape) != 2 or (cols is not None and a.shape[1] != cols):
        raise ValueError(f"{name} has shape {a.shape}" + (f", {cols} columns are needed" if cols is not None else ""))
    m, k = a.shape
    if stride is None:
        return kind, m, k, k
    if stride < k:
        raise ValueError(f"{name}: rows of {k} at a stride of {stride}")
    _within(name, a, m, k, stride)
    return kind, m, k, stride


def _ids(which, rows):
    if which.dtype != np.int32:
        raise TypeError(f"row numbers must be int32, not {which.dtype}")
    if which.shape[0] != rows:
        raise ValueError(f"{which.shape[0]} row numbers for {rows} rows")


class _Kept(threading.local):
    """a thread's workspaces by (device, stream)"""

    def __init__(self):
        self.blocks = _Blocks()
        with _threads_lock:
            _threads.add(self.blocks)


class _Blocks(dict):
    __hash__ = object.__hash__                            # one of its thread, whatever it holds


_threads, _threads_lock = weakref.WeakSet(), threading.RLock()
_kept = _Kept()


def _stream_ends(stream):
    """a stream that ends takes every thread's workspace for it along: the next stream may get its handle"""
    with _threads_lock:
        for blocks in list(_threads):
            for key in [k for k in list(blocks) if k[1] == stream]:
                blocks.pop(key, None)


dev.Stream.ends.append(_stream_ends)


class _Block:
    """a workspace's memory, apart from the arrays' cache: a block there may still be in use by the work of another
    stream. Freeing it waits for the device."""
    __slots__ = ("ptr", "nbytes")

    def __init__(self, n):
        self.ptr, self.nbytes = dev.CACHE.alloc(n), n

    def __del__(self):
        try:
            lib().spa_free(self.ptr)
        except Exception:
            pass


def _not_captured(stream, what):
    """a graph keeps the addresses of its capture, so what it uses has to be the caller's"""
    if stream is not None:
        yes = ctypes.c_int()
        check(lib().spa_stream_is_capturing(stream, ctypes.byref(yes)))
        if yes.value:
            raise ValueError(f"a call that is captured needs its {what} given")


def _scratch(n, work, stream):
    """the call's workspace: the one given, or this thread's own for the device and stream, kept for its next calls
    there (a captured call's is given: the graph keeps its address). One that has to grow waits for the stream once, so that work still queued on the old block is done.
    -> (what keeps it alive, pointer, bytes)"""
    if not n:
        return None, None, 0
    if work is None:
        _not_captured(stream, "workspace (work)")
        blocks, key = _kept.blocks, (dev.current_device(), stream)
        work = blocks.get(key)
        if work is None or work.nbytes < n:
            if work is not None:
                check(lib().spa_stream_synchronize(stream))
                del blocks[key], work
            work = blocks[key] = _Block(max(n, 1 << 20))
    return work, work.ptr, work.nbytes


def release():
    """frees this thread's workspaces, after waiting for the work of their devices (not for their streams, which may
    have ended). To be called before a stream that is not a device.Stream ends, if calls were made on it."""
    blocks, here = _kept.blocks, dev.current_device()
    try:
        for d in sorted({d for d, _ in list(blocks)}):
            dev.set_device(d)
            check(lib().spa_device_synchronize())
    finally:
        dev.set_device(here)
        blocks.clear()


def _out(name, out, m, n, dtype, stride, stream):
    if out is None:
        if stride is not None:
            raise ValueError(f"a stride of {name} needs its array")
        _not_captured(stream, f"result ({name})")
        return dev.DeviceArray((m, n), dtype), n
    if out.dtype != dtype or out.shape != (m, n):
        raise ValueError(f"{name} is {out.shape} {out.dtype}, ({m}, {n}) {dtype} is needed")
    if stride is not None and stride < n:
        raise ValueError(f"{name}: rows of {n} at a stride of {stride}")
    if stride is not None:
        _within(name, out, m, n, stride)
    return out, n if stride is None else stride


def project(x, w, adapters=None, which=None, out=None, x_stride=None, out_stride=None, work=None, stream=None):
    """x (rows, w.cols) -> (rows, w.rows): x W^T, plus for each row r the adapter which[r] (int32; numbers
    outside the pool: none)"""
    kind, m, _, ld = _rows("x", x, x_stride, w.cols)
    a = b = scale = ids = None
    pool = rank = 0
    if adapters is not None:
        if which is None:
            raise ValueError("adapters need the number of each row's adapter")
        if adapters.a.dtype != x.dtype or adapters.a.shape[2] != w.cols or adapters.b.shape[1] != w.rows:
            raise ValueError(f"adapters of {adapters.a.dtype} {adapters.a.shape}, {adapters.b.shape} beside {x.dtype} inputs "
                             f"and a {w.rows} x {w.cols} projection")
        _ids(which, m)
        if which.size != m:
            raise ValueError(f"adapters' numbers of shape {which.shape}: one for each of the {m} rows")
        a, b, scale, ids, pool, rank = adapters.a.ptr, adapters.b.ptr, adapters.scale.ptr, which.ptr, adapters.count, adapters.rank
    out, ldo = _out("out", out, m, w.rows, x.dtype, out_stride, stream)
    L = lib()
    keep, p, n = _scratch(L.spa_project_work_bytes(w.type, w.rows, w.cols, kind, m, pool, rank), work, stream)
    check(L.spa_project(w.type, w.data.ptr, w.rows, w.cols, kind, x.ptr, m, ld, out.ptr, ldo, a, b, scale, pool, rank, ids,
                        p, n, stream))
    return out


def _pair(gate, up, act):
    if (gate.type, gate.rows, gate.cols) != (up.type, up.rows, up.cols):
        raise ValueError(f"gate is type {gate.type} {gate.rows} x {gate.cols}, up type {up.type} {up.rows} x {up.cols}")
    if act not in ACT:
        raise ValueError(f"unknown activation {act!r}: {sorted(ACT)}")
    return ACT[act]


def gated(x, gate, up, act="silu", out=None, x_stride=None, out_stride=None, work=None, stream=None):
    """x (rows, cols) -> act(x gate^T) * (x up^T), (rows, gate.rows); act "silu" or "gelu" (tanh form)"""
    act = _pair(gate, up, act)
    kind, m, _, ld = _rows("x", x, x_stride, gate.cols)
    out, ldo = _out("out", out, m, gate.rows, x.dtype, out_stride, stream)
    L = lib()
    keep, p, n = _scratch(L.spa_gated_work_bytes(gate.type, gate.rows, gate.cols, kind, m), work, stream)
    check(L.spa_gated(gate.type, gate.data.ptr, up.data.ptr, gate.rows, gate.cols, kind, x.ptr, m, ld, act, out.ptr, ldo, p, n,
                      stream))
    return out


def gated_backward(x, gate, up, dh, act="silu", dx=None, dgate=None, dup=None, x_stride=None, dh_stride=None, dx_stride=None,
                   work=None, stream=None):
    """the gradients of gated() from dh (rows, gate.rows): written to the arrays given, dx (rows, cols) and / or
    both of dgate and dup (gate.rows, cols; weights of x's own type only). With none given dx is made.
    -> (dx, dgate, dup)"""
    act = _pair(gate, up, act)
    kind, m, k, ld = _rows("x", x, x_stride, gate.cols)
    _, mh, _, ldh = _rows("dh", dh, dh_stride, gate.rows)
    if mh != m or dh.dtype != x.dtype:
        raise ValueError(f"dh is {dh.shape} {dh.dtype} for x {x.shape} {x.dtype}")
    if (dgate is None) != (dup is None):
        raise ValueError("both matrices' gradients or neither")
    ldx = k
    if dx is not None or dgate is None:
        dx, ldx = _out("dx", dx, m, k, x.dtype, dx_stride, stream)
    if dgate is not None:
        dgate, _ = _out("dgate", dgate, gate.rows, k, x.dtype, None, stream)
        dup, _ = _out("dup", dup, gate.rows, k, x.dtype, None, stream)
    L = lib()
    keep, p, n = _scratch(L.spa_gated_backward_work_bytes(gate.type, gate.rows, k, kind, m, dx is not None, dgate is not None), work, stream)
    check(L.spa_gated_backward(gate.type, gate.data.ptr, up.data.ptr, gate.rows, k, kind, x.ptr, m, ld, act, dh.ptr, ldh,
                               None if dx is None else dx.ptr, ldx, None if dgate is None else dgate.ptr,
                               None if dup is None else dup.ptr, p, n, stream))
    return dx, dgate, dup


def add_squares(x, sums, counts, which=None, x_stride=None, work=None, stream=None):
    """x (rows, cols), float32 too: adds the rows' squares to sums (experts, cols) float32 and their numbers to
    counts (experts,) int64. which (rows, each) int32 holds the experts of each row; without it there is one sum
    over all rows. An importance matrix is sums / counts, and 1 for an expert without rows, as
    imatrix.load reads "in_sum2" and "counts"; imatrix.write_dat makes a file of it."""
    kind, m, k, ld = _rows("x", x, x_stride)
    experts = each = 0
    if which is not None:
        _ids(which, m)
        experts, each = counts.size, (which.size // m if m else 1)
    if sums.dtype != np.float32 or counts.dtype != np.int64 or sums.size != counts.size * k or (which is None and counts.size != 1):
        raise ValueError(f"sums {sums.shape} {sums.dtype}, counts {counts.shape} {counts.dtype} for {k} columns")
    L = lib()
    keep, p, n = _scratch(L.spa_add_squares_work_bytes(m, k, experts), work, stream)
    check(L.spa_add_squares(x.ptr, kind, m, k, ld, None if which is None else which.ptr, each, experts, sums.ptr, counts.ptr,
                            p, n, stream))
    return sums, counts
