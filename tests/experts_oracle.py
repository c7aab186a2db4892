"""Routing, 4-bit blocks and products by expert from their definitions, in float64 with numpy on the host."""
import numpy as np

GRID = np.array([0, .5, 1, 1.5, 2, 3, 4, 6])
F32, BF16, F16 = np.float32, np.uint16, np.float16
#: half a step of a type, relative to the value
HALF = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}
#: half of the least step
LEAST = {BF16: 2.0 ** -134, F16: 2.0 ** -25, F32: 2.0 ** -150}


def rng(*key):
    return np.random.Generator(np.random.PCG64(list(key)))


def store(v, kind):
    """float64 -> a type's numbers (bf16 as its bits), to nearest even"""
    with np.errstate(over="ignore"):
        if kind is not BF16:
            return v.astype(kind)
        f = v.astype(np.float32)
    b = f.view(np.uint32)
    r = ((b.astype(np.uint64) + 0x7fff + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isfinite(f), r, (b >> 16).astype(np.uint16) | np.isnan(f) * np.uint16(0x40)).astype(np.uint16)


def wide(a):
    if a.dtype == np.uint16:
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


# ------------------------------------------------------------------------------------------ routing

def softmax(l):
    with np.errstate(invalid="ignore", over="ignore"):
        p = np.exp(l - l.max(1, keepdims=True))
        return p / p.sum(1, keepdims=True)


def sigmoid(l):
    with np.errstate(over="ignore"):
        return 1 / (1 + np.exp(-l))


def choose(l, each, score, bias=None, groups=1, keep=1, best=2):
    """which (rows, each), -1 where none is left"""
    m, e = l.shape
    with np.errstate(invalid="ignore"):
        key = l.copy()
        if bias is not None or groups > 1:
            key = np.where(l == -np.inf, -np.inf, softmax(l) if score == "softmax" else sigmoid(l))
            if bias is not None:
                key = key + bias.astype(np.float64)
    key[np.isnan(key)] = np.inf                      # above all: no test has both
    if groups > 1:
        runs = key.reshape(m, groups, -1)
        top = -np.sort(-runs, axis=2)[:, :, :best].sum(2)
        kept = np.argsort(-top, axis=1, kind="stable")[:, :keep]
        mask = np.zeros((m, groups), bool)
        np.put_along_axis(mask, kept, True, 1)
        key = np.where(np.repeat(mask, e // groups, 1), key, -np.inf)
    which = np.argsort(-key, axis=1, kind="stable")[:, :each]
    return np.where(np.take_along_axis(key, which, 1) == -np.inf, -1, which).astype(np.int32)


def log_scores(l, score):
    """the scores' logarithms, up to a number of their own for each row"""
    return l if score == "softmax" else -np.logaddexp(0, -l)


def shares(l, which, score):
    """the chosen scores over their sum"""
    t = np.where(which < 0, -np.inf, np.take_along_axis(log_scores(l, score), np.maximum(which, 0), 1))
    top = t.max(1, keepdims=True)
    v = np.exp(t - np.where(np.isfinite(top), top, 0))
    s = v.sum(1, keepdims=True)
    return np.where(which < 0, 0, v / np.where(s == 0, 1, s))


def weights(l, which, score, renorm, scale):
    if renorm:
        return scale * shares(l, which, score)
    s = softmax(l) if score == "softmax" else sigmoid(l)
    return np.where(which < 0, 0, scale * np.take_along_axis(s, np.maximum(which, 0), 1))


def route_backward(l, which, dw, score, renorm, scale):
    """-> (gradient, the sum of the magnitudes that it is made of)"""
    m, e = l.shape
    valid = (which >= 0) & (which < e)
    at = np.where(valid, which, -1)
    s = softmax(l) if score == "softmax" else sigmoid(l)
    p = np.where(valid, np.take_along_axis(s, np.maximum(at, 0), 1), 0)
    dw = np.where(valid, dw, 0).astype(np.float64)
    if renorm:
        q = shares(l, at, score)
        a, t = scale * q * (dw - (q * dw).sum(1, keepdims=True)), scale * q * (abs(dw) + (q * abs(dw)).sum(1, keepdims=True))
    else:
        a = scale * p * dw
        t = abs(a)
    out, size = np.zeros((m, e)), np.zeros((m, e))
    for j in range(which.shape[1]):
        slope = 1 - p[:, j] if score == "sigmoid" else 1
        np.add.at(out, (np.arange(m)[valid[:, j]], at[valid[:, j], j]), (a[:, j] * slope)[valid[:, j]])
        np.add.at(size, (np.arange(m)[valid[:, j]], at[valid[:, j], j]), t[valid[:, j], j])
    if score == "softmax" and not renorm:
        out -= s * a.sum(1, keepdims=True)
        size += s * t.sum(1, keepdims=True)
    return out, size


def by_expert(which, experts):
    flat = which.reshape(-1)
    key = np.where((flat >= 0) & (flat < experts), flat, experts)
    order = np.argsort(key, kind="stable").astype(np.int32)
    starts = np.concatenate([[0], np.cumsum(np.bincount(key, minlength=experts + 1))])[:experts + 1].astype(np.int32)
    return order, starts


# ------------------------------------------------------------------------------------------ 4 bits

def quantize(x):
    """rows -> (codes, scales) of whole runs of eight blocks"""
    m, k = x.shape
    b = np.zeros((m, -(-k // 256) * 256))
    b[:, :k] = x
    b = b.reshape(m, -1, 32)
    top = abs(b).max(2)
    fine = np.isfinite(top)
    e = np.maximum(np.frexp(np.where(fine & (top > 0), top, 2.0 ** -200))[1] - 3, -127)
    v = np.where(fine[:, :, None], b, 0) / 2.0 ** e[:, :, None]
    size = abs(v)
    code = np.zeros(v.shape, np.uint8)
    for c in range(1, 8):                            # past the middle of two neighbours, or on it beside an even upper one
        half = (GRID[c - 1] + GRID[c]) / 2
        code[(size > half) | ((size == half) & (c % 2 == 0))] = c
    code |= (np.signbit(v) & fine[:, :, None]).astype(np.uint8) << 3
    codes = (code[:, :, :16] | code[:, :, 16:] << 4).reshape(m, -1)
    return codes, np.where(fine, e + 127, 255).astype(np.uint8)


def values(codes, scales, cols):
    m = len(codes)
    b = codes.reshape(m, -1, 16)
    c = np.concatenate([b & 15, b >> 4], 2)
    v = GRID[c & 7] * np.where(c >> 3, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return (v * s.reshape(m, -1)[:, :, None]).reshape(m, -1)[:, :cols]


def act(g, name):
    with np.errstate(over="ignore"):
        if name == "silu":
            return g / (1 + np.exp(-g))
        return 0.5 * g * (1 + np.tanh(np.sqrt(2 / np.pi) * (g + 0.044715 * g ** 3)))
