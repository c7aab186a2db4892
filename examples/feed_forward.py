"""A feed-forward block from calibration to serving, on one GPU:

  1. a text's activations go through the BF16 block, and the squares of each matrix's inputs are gathered;
  2. with them as the importance the three matrices are quantized, and stay in device memory as blocks;
  3. the quantized block is compared with the base (with the importance, and without it);
  4. one gradient step moves the base's gate and up matrices towards a block that they differ from;
  5. a decoding batch goes through the quantized block, each request with a low-rank adapter of its own.

    python examples/feed_forward.py [--cols 1024] [--inner 4096] [--tokens 2048]
"""
import argparse
import os
import sys

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from seedpack_amd import device as dev  # noqa: E402
from seedpack_amd import linear, synth  # noqa: E402
from seedpack_amd.gpuquant import GPUQuant  # noqa: E402
from seedpack_amd.requant import BY_NAME  # noqa: E402

Q4_K = BY_NAME["Q4_K"]


def bits(v):
    """float32 -> bf16 bits, to nearest even"""
    b = np.ascontiguousarray(v, np.float32).view(np.uint32)
    return ((b + 0x7fff + ((b >> 16) & 1)) >> 16).astype(np.uint16)


def floats(a):
    return synth.bf16_to_f32(a.to_host()).reshape(a.shape)


def importance(rows, chunk=512):
    """the mean square of each column, gathered a chunk of rows at a time as a calibration run would"""
    m, k = rows.shape
    sums, counts = dev.DeviceArray((1, k), np.float32).zero(), dev.DeviceArray((1,), np.int64).zero()
    for r in range(0, m, chunk):
        n = min(chunk, m - r)
        linear.add_squares(rows.view(2 * r * k, (n, k), np.uint16), sums, counts)
    return sums.to_host()[0] / np.float32(counts.to_host()[0])


def block(x, gate, up, down, adapters=None, which=None):
    return linear.project(linear.gated(x, gate, up), down, adapters, which)


def run(cols=1024, inner=4096, tokens=2048, requests=24, seed=1):
    g = np.random.Generator(np.random.PCG64(seed))
    shapes = {"gate": (inner, cols), "up": (inner, cols), "down": (cols, inner)}
    host = {name: synth.normal_bf16(g, s, 0.03, outlier_frac=0.001) for name, s in shapes.items()}
    base = {name: linear.Weight(linear.BF16, dev.DeviceArray.from_host(w.reshape(-1)), *shapes[name]) for name, w in host.items()}
    size = np.exp(g.normal(0, 1, cols))
    text = lambda n: dev.DeviceArray.from_host(bits(g.normal(0, 1, (n, cols)) * size))

    x = text(tokens)                                                                         # 1
    h = linear.gated(x, base["gate"], base["up"])
    imx = {"gate": importance(x), "up": importance(x), "down": importance(h)}

    def quantized(imatrices):                                                                # 2
        out = {}
        for name, (n, k) in shapes.items():
            blocks = GPUQuant().quantize_tensors(Q4_K, [(host[name].reshape(-1), k)], [imatrices.get(name)], device=True)[0]
            out[name] = linear.Weight(Q4_K, blocks, n, k)
        return out

    held = text(512)                                                                         # 3
    want = floats(block(held, **base))
    off = lambda y: float(np.linalg.norm(floats(y) - want) / np.linalg.norm(want))
    quant = quantized(imx)
    error, error_plain = off(block(held, **quant)), off(block(held, **quantized({})))

    few = text(256)                                                                          # 4
    other = {n: linear.Weight(linear.BF16, dev.DeviceArray.from_host(bits(synth.bf16_to_f32(host[n]).reshape(shapes[n]) +
                              g.normal(0, 0.01, shapes[n]))), *shapes[n]) for n in ("gate", "up")}
    target = floats(linear.gated(few, other["gate"], other["up"]))
    loss = lambda gate, up: 0.5 * float(((floats(linear.gated(few, gate, up)) - target) ** 2).mean())
    apart = floats(linear.gated(few, base["gate"], base["up"])) - target
    dh = dev.DeviceArray.from_host(bits(apart))
    grads = {n: dev.DeviceArray(shapes[n], np.uint16) for n in ("gate", "up")}
    linear.gated_backward(few, base["gate"], base["up"], dh, dgate=grads["gate"], dup=grads["up"])
    wide = {n: floats(grads[n]) for n in grads}
    # the step that would lower half the sum of squares by a tenth were it linear along the gradient
    rate = 0.1 * 0.5 * float((apart ** 2).sum()) / sum(float((v.astype(np.float64) ** 2).sum()) for v in wide.values())
    stepped = {n: linear.Weight(linear.BF16, dev.DeviceArray.from_host(bits(synth.bf16_to_f32(host[n]).reshape(shapes[n]) - rate * wide[n])),
                                *shapes[n]) for n in grads}
    before, after = loss(base["gate"], base["up"]), loss(stepped["gate"], stepped["up"])

    rank, pool = 16, 6                                                                       # 5
    a = bits(g.normal(0, 1, (pool, rank, inner)) / np.sqrt(inner))
    b = bits(g.normal(0, 0.05, (pool, cols, rank)))
    adapters = linear.Adapters(dev.DeviceArray.from_host(a), dev.DeviceArray.from_host(b), dev.DeviceArray.from_host(np.ones(pool, np.float32)))
    which = dev.DeviceArray.from_host(g.integers(-1, pool, requests).astype(np.int32))
    batch = text(requests)
    plain, tuned = floats(block(batch, **quant)), floats(block(batch, **quant, adapters=adapters, which=which))
    moved = np.abs(tuned - plain).max(1) > 0
    return {"error": error, "error_plain": error_plain, "before": before, "after": after,
            "moved": moved.tolist(), "which": which.to_host().tolist()}


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--cols", type=int, default=1024)
    ap.add_argument("--inner", type=int, default=4096)
    ap.add_argument("--tokens", type=int, default=2048)
    a = ap.parse_args()
    r = run(a.cols, a.inner, a.tokens)
    print(f"Q4_K block against its base: {r['error']:.4f} off with the gathered importance, {r['error_plain']:.4f} without")
    print(f"one gradient step: loss {r['before']:.6f} -> {r['after']:.6f}")
    print(f"decoding batch: {sum(r['moved'])} of {len(r['moved'])} requests have an adapter")


if __name__ == "__main__":
    main()
