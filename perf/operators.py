"""What the speed of the products with packed weights is measured on: the calls that a program makes
which applies a model's regrown tensors, tunes on its base, or gathers the importance its quants are
made with.

  squares         the column sums of squares of a matrix's inputs, whole or per expert: an importance
                  matrix as it is gathered, one call per matrix and chunk of text
  project         a shared projection with the low-rank adapters of the requests in the batch
  gated           the gated half of a feed-forward block: both projections, the activation, the product
  gated_backward  its gradients: with those of the weights (tuning on the base), or of the inputs alone
                  (through a frozen quant)

Weights are BF16 or F16 matrices or GGUF blocks, row-major, in device memory.
"""
import math

import torch

own = False

#: ggml type ids, weights per block, bytes per block
TYPES = {"F16": (1, 1, 2), "BF16": (30, 1, 2), "Q8_0": (8, 32, 34), "Q4_K": (12, 256, 144), "Q6_K": (14, 256, 210)}
KIND = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ------------------------------------------------------------------------------------------ the cases

def _squares(rows, cols, x="bf16", experts=0, each=1):
    return {"op": "squares", "rows": rows, "cols": cols, "x": x, "experts": experts, "each": each}


def _project(rows, n, cols, quant, x="bf16", pool=0, rank=0):
    return {"op": "project", "rows": rows, "n": n, "cols": cols, "quant": quant, "x": x, "pool": pool, "rank": rank}


def _gated(rows, n, cols, quant, x="bf16", act="silu"):
    return {"op": "gated", "rows": rows, "n": n, "cols": cols, "quant": quant, "x": x, "act": act}


def listed():
    def named(name, case):
        return dict(case, name=name)

    return [
        # one chunk of a calibration text at the input of an attention matrix: the smallest call
        named("squares-chunk", _squares(512, 4096)),
        # the tokens of a long batch, each sent to two of 64 experts, in the order they came in
        named("squares-experts", _squares(16384, 4096, experts=64, each=2)),
        # the inputs of a feed-forward block's last matrix over a whole batch, in 32 bits
        named("squares-wide", _squares(16384, 12288, x="f32")),
        # one new token of one request with a fine tune of its own: latency is all
        named("project-token", _project(1, 4096, 4096, "Q4_K", pool=8, rank=16)),
        # a decoding batch of 32 requests over 16 fine tunes
        named("project-batch", _project(32, 12288, 4096, "Q8_0", pool=16, rank=16)),
        # the vocabulary's projection for three tokens: the largest matrix of a small model
        named("project-vocabulary", _project(3, 151936, 1024, "Q6_K")),
        # the prompts of four requests behind one another
        named("project-prompts", _project(2053, 4096, 12288, "Q4_K", pool=4, rank=64)),
        # ragged in every size: rows, outputs, columns and rank, in half precision
        named("project-ragged", _project(517, 2053, 3584, "F16", x="f16", pool=5, rank=12)),
        # one new token through a quantized block
        named("gated-token", _gated(1, 12288, 4096, "Q4_K")),
        # a batch of text through the base's block
        named("gated-text", _gated(4096, 12288, 4096, "BF16")),
        # a tuning step on the base
        named("gated_backward-base", dict(_gated(4096, 12288, 4096, "BF16"), op="gated_backward")),
        # the gradient that passes a frozen 8-bit block on its way to the layers below
        named("gated_backward-frozen", dict(_gated(1000, 12288, 4096, "Q8_0", act="gelu"), op="gated_backward")),
    ]


def _spread(rng, least, most):
    """a whole number, even over the logarithm"""
    return min(most, max(least, round(math.exp(rng.uniform(math.log(least), math.log(most + 1))))))


def draw(rng):
    op = rng.choices(["squares", "project", "gated", "gated_backward"], [25, 40, 20, 15])[0]
    if op == "squares":
        experts = rng.choice([0, 0, _spread(rng, 2, 64)])
        rows, cols = _spread(rng, 1, 32768), _spread(rng, 33, 12288)
        return _squares(min(rows, (3 << 26) // cols), cols, rng.choice(["bf16", "bf16", "f16", "f32"]), experts,
                        rng.choice([1, 2]) if experts else 1)
    x, quant = rng.choice([("bf16", "BF16"), ("f16", "F16"), ("bf16", "Q8_0"), ("bf16", "Q4_K"), ("bf16", "Q6_K"),
                           ("f16", "Q4_K")])
    qk = TYPES[quant][1]
    cols = qk * _spread(rng, max(1, 64 // qk), 12288 // qk)
    n = _spread(rng, 33, 16384)
    rows = min(_spread(rng, 1, 4096), max(1, int(1e11 / (cols * n))))
    if op == "project":
        pool = rng.choice([0, _spread(rng, 1, 16)])
        return _project(rows, n, cols, quant, x, pool, _spread(rng, 1, 64) if pool else 0)
    return dict(_gated(rows, n, cols, quant, x, rng.choice(["silu", "gelu"])), op=op)


# ------------------------------------------------------------------------------------------ inputs

def _q8_0(w):
    b = w.view(-1, 32)
    d = (b.abs().amax(1, True) / 127).half()
    q = torch.round(b / d.float().clamp(min=1e-7)).clamp(-127, 127).to(torch.int8)
    return torch.cat([d.view(torch.uint8), q.view(torch.uint8)], 1)


def _q4_k(w):
    b = w.view(-1, 8, 32)
    low = (-b.amin(2)).clamp(min=0)
    step = (b.amax(2) + low) / 15
    d, dm = (step.amax(1, True) / 63).half(), (low.amax(1, True) / 63).half()
    sc = torch.round(step / d.float().clamp(min=1e-7)).clamp(0, 63)
    mn = torch.round(low / dm.float().clamp(min=1e-7)).clamp(0, 63)
    q = (b + (dm.float() * mn)[:, :, None]) / (d.float() * sc).clamp(min=1e-7)[:, :, None]
    q = torch.round(q).clamp(0, 15).to(torch.uint8).view(-1, 4, 2, 32)
    sc, mn = sc.to(torch.uint8), mn.to(torch.uint8)
    head = [sc[:, :4] | (sc[:, 4:] >> 4 << 6), mn[:, :4] | (mn[:, 4:] >> 4 << 6), (sc[:, 4:] & 15) | ((mn[:, 4:] & 15) << 4)]
    return torch.cat([d.view(torch.uint8), dm.view(torch.uint8), *head, (q[:, :, 0] | q[:, :, 1] << 4).flatten(1)], 1)


def _q6_k(w):
    b = w.view(-1, 16, 16)
    step = b.abs().amax(2) / 31
    d = (step.amax(1, True) / 127).half()
    sc = torch.round(step / d.float().clamp(min=1e-7)).clamp(0, 127)
    q = torch.round(b / (d.float() * sc).clamp(min=1e-7)[:, :, None]).clamp(-32, 31) + 32
    q = q.to(torch.uint8).view(-1, 2, 4, 32)
    lo = (q[:, :, :2] & 15) | ((q[:, :, 2:] & 15) << 4)
    hi = q[:, :, 0] >> 4 | q[:, :, 1] >> 4 << 2 | q[:, :, 2] >> 4 << 4 | q[:, :, 3] >> 4 << 6
    return torch.cat([lo.flatten(1), hi.flatten(1), sc.to(torch.uint8), d.view(torch.uint8)], 1)


def _stored(g, quant, n, cols):
    """a matrix of n rows as it lies in memory: normal weights with a few large ones"""
    w = torch.randn(n, cols, generator=g, device="cuda").mul_(0.02)
    w[torch.rand(n, cols, generator=g, device="cuda") < 1e-3] *= 8
    if quant in ("F16", "BF16"):
        return w.to(KIND[quant.lower()])
    return {"Q8_0": _q8_0, "Q4_K": _q4_k, "Q6_K": _q6_k}[quant](w).reshape(n, -1)


def _rows(g, rows, cols, x):
    """activations: columns of unlike size, a few of them far larger than the rest"""
    size = torch.randn(cols, generator=g, device="cuda").mul_(0.5).exp_()
    size[torch.rand(cols, generator=g, device="cuda") < 2e-3] *= 20
    return (torch.randn(rows, cols, generator=g, device="cuda") * size).to(KIND[x])


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op, rows, cols, x = case["op"], case["rows"], case["cols"], case["x"]
    s = dict(case, x=_rows(g, rows, cols, x))
    if op == "squares":
        e = case["experts"]
        s["sums"] = torch.zeros(max(e, 1), cols, device="cuda")
        s["counts"] = torch.zeros(max(e, 1), dtype=torch.int64, device="cuda")
        if e:   # unlike experts: the first of them get most rows
            at = torch.rand(rows, case["each"], generator=g, device="cuda").square_() * e
            s["which"] = at.to(torch.int32).clamp(max=e - 1)
        return s
    n, quant = case["n"], case["quant"]
    if op == "project":
        s["w"] = _stored(g, quant, n, cols)
        if case["pool"]:
            p, r = case["pool"], case["rank"]
            s["a"] = (torch.randn(p, r, cols, generator=g, device="cuda") / math.sqrt(cols)).to(KIND[x])
            s["b"] = torch.randn(p, n, r, generator=g, device="cuda").mul_(0.05).to(KIND[x])
            s["scale"] = torch.rand(p, generator=g, device="cuda") + 0.5
            which = torch.randint(-1, p, (rows,), generator=g, device="cuda", dtype=torch.int32)
            # decoding rows come in any order, the rows of prompts one request behind another
            s["which"] = torch.sort(which).values.int() if rows > 256 else which.clamp(min=0 if rows == 1 else -1)
        return s
    s["gate"], s["up"] = _stored(g, quant, n, cols), _stored(g, quant, n, cols)
    if op == "gated_backward":
        size = torch.randn(rows, 1, generator=g, device="cuda").exp_() * 1e-2
        s["dh"] = (torch.randn(rows, n, generator=g, device="cuda") * size).to(KIND[x])
    return s


# ------------------------------------------------------------------------------------------ one pass

def _wide(w, quant, cols):
    """the weights of a stored matrix, in 32 bits"""
    if quant in ("F16", "BF16"):
        return w.float()
    n, b = len(w), w.reshape(-1, TYPES[quant][2])
    half = lambda o: b[:, o:o + 2].contiguous().view(torch.float16).float()            # (blocks, 1)
    if quant == "Q8_0":
        return (half(0) * b[:, 2:].contiguous().view(torch.int8)).view(n, cols)
    if quant == "Q4_K":
        s, q = b[:, 4:16], b[:, 16:].view(-1, 4, 1, 32)
        sc = torch.cat([s[:, :4] & 63, (s[:, 8:] & 15) | (s[:, :4] >> 6 << 4)], 1)
        mn = torch.cat([s[:, 4:8] & 63, (s[:, 8:] >> 4) | (s[:, 4:8] >> 6 << 4)], 1)
        q = torch.cat([q & 15, q >> 4], 2).view(-1, 8, 32)
        return ((half(0) * sc)[:, :, None] * q - (half(2) * mn)[:, :, None]).view(n, cols)
    lo, hi = b[:, :128].view(-1, 2, 2, 32), b[:, 128:192].view(-1, 2, 1, 32)
    q = torch.cat([lo & 15, lo >> 4], 2) | (torch.cat([hi, hi >> 2, hi >> 4, hi >> 6], 2) & 3) << 4
    sc = half(208) * b[:, 192:208].contiguous().view(torch.int8)
    return (sc[:, :, None] * (q.view(-1, 16, 16).float() - 32)).view(n, cols)


def _act(g, act):
    """the activation and its derivative"""
    if act == "silu":
        p = 1 / (1 + torch.exp(-g))
        return g * p, p * (1 + g * (1 - p))
    t = torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * g * g)


def _plain(s):
    op, kind = s["op"], s["x"].dtype
    x = s["x"].float()
    if op == "squares":
        if not s["experts"]:
            return {"sums": s["sums"] + (x * x).sum(0, True), "counts": s["counts"] + len(x)}
        hit = (s["which"][:, :, None] == torch.arange(s["experts"], device="cuda")).sum(1)
        return {"sums": s["sums"] + hit.float().t() @ (x * x), "counts": s["counts"] + hit.sum(0)}
    if op == "project":
        y = x @ _wide(s["w"], s["quant"], s["cols"]).t()
        if s["pool"]:
            p, r = s["pool"], s["rank"]
            z = (x @ s["a"].float().view(p * r, -1).t()).view(-1, p, r)
            mine = (s["which"][:, None] == torch.arange(p, device="cuda")) * s["scale"]
            y = y + (z * mine[:, :, None]).view(-1, p * r) @ s["b"].float().transpose(1, 2).reshape(p * r, -1)
        return y.to(kind)
    wg, wu = _wide(s["gate"], s["quant"], s["cols"]), _wide(s["up"], s["quant"], s["cols"])
    u = x @ wu.t()
    a, da = _act(x @ wg.t(), s["act"])
    if op == "gated":
        return (a * u).to(kind)
    dh = s["dh"].float()
    dg, du = dh * u * da, dh * a
    grads = {"dx": (dg @ wg + du @ wu).to(kind)}
    if s["quant"] in ("F16", "BF16"):
        grads |= {"dgate": (dg.t() @ x).to(kind), "dup": (du.t() @ x).to(kind)}
    return grads


def run(s):
    if not own:
        return _plain(s)
    import numpy as np
    from seedpack_amd import device as dev, linear

    names = {torch.bfloat16: np.uint16, torch.float16: np.float16, torch.float32: np.float32, torch.uint8: np.uint8,
             torch.int32: np.int32, torch.int64: np.int64}

    def array(t):
        return dev.DeviceArray(t.shape, names[t.dtype], ptr=t.data_ptr(), owner=t)

    op, x = s["op"], array(s["x"])
    stream = torch.cuda.current_stream().cuda_stream or None
    if op == "squares":
        # a program keeps its sums; here each pass returns its own, as the plain form does
        sums, counts = s["sums"].clone(), s["counts"].clone()
        linear.add_squares(x, array(sums), array(counts), array(s["which"]) if s["experts"] else None, stream=stream)
        return {"sums": sums, "counts": counts}
    weight = lambda t: linear.Weight(TYPES[s["quant"]][0], array(t), s["n"], s["cols"])
    if op == "project":
        y = torch.empty(s["rows"], s["n"], dtype=s["x"].dtype, device="cuda")
        adapters = linear.Adapters(array(s["a"]), array(s["b"]), array(s["scale"])) if s["pool"] else None
        linear.project(x, weight(s["w"]), adapters, array(s["which"]) if s["pool"] else None, out=array(y), stream=stream)
        return y
    if op == "gated":
        h = torch.empty(s["rows"], s["n"], dtype=s["x"].dtype, device="cuda")
        linear.gated(x, weight(s["gate"]), weight(s["up"]), s["act"], out=array(h), stream=stream)
        return h
    grads = {"dx": torch.empty_like(s["x"])}
    if s["quant"] in ("F16", "BF16"):
        grads |= {"dgate": torch.empty_like(s["gate"]), "dup": torch.empty_like(s["up"])}
    linear.gated_backward(x, weight(s["gate"]), weight(s["up"]), array(s["dh"]), s["act"],
                          **{k: array(v) for k, v in grads.items()}, stream=stream)
    return grads


# ------------------------------------------------------------------------------------------ its work

def work(case):
    op, m, k = case["op"], case["rows"], case["cols"]
    if op == "squares":
        e = max(1, case["experts"])
        ids = 4 * m * case["each"] if case["experts"] else 0
        return {"bytes": m * k * KIND[case["x"]].itemsize + ids + 8 * e * k, "flops": 2 * m * k * case["each"]}
    n, (_, qk, bs) = case["n"], TYPES[case["quant"]]
    w = n * k // qk * bs
    if op == "project":
        used, r = min(case["pool"], m), case["rank"]
        return {"bytes": w + 2 * m * (n + k) + 2 * used * r * (n + k), "flops": 2 * m * n * k + 2 * m * r * (n + k)}
    if op == "gated":
        return {"bytes": 2 * w + 2 * m * (n + k), "flops": 4 * m * n * k}
    tuned = case["quant"] in ("F16", "BF16")
    return {"bytes": 2 * w * (2 if tuned else 1) + 2 * m * (n + 2 * k), "flops": (12 if tuned else 8) * m * n * k}


# ------------------------------------------------------------------------------------------ in 64 bits

def _weights64(w, quant, cols):
    """the weights of a stored matrix by the block's definition, a weight at a time: its code's bits, then
    scale and offset by its index in the block"""
    if quant in ("F16", "BF16"):
        return w.double()
    _, qk, bs = TYPES[quant]
    b = w.reshape(-1, bs).int()
    i = torch.arange(qk, device="cuda")

    def half(at):                                    # binary16 from its two bytes, by sign, exponent, mantissa
        v = b[:, at] | b[:, at + 1] << 8
        e, m = (v >> 10 & 31).double(), (v & 1023).double()
        size = torch.where(e > 0, torch.exp2(e - 25) * (1024 + m), torch.exp2(torch.tensor(-24.0, device="cuda").double()) * m)
        return (size * (1 - 2 * (v >> 15)))[:, None]

    signed = lambda v: (v ^ 128) - 128
    if quant == "Q8_0":
        out = half(0) * signed(b[:, 2 + i])
    elif quant == "Q4_K":
        sub = i // 32
        code = b[:, 16 + 32 * (sub // 2) + i % 32] >> (4 * (sub % 2)) & 15
        s, t = b[:, 4 + sub % 4], b[:, 8 + sub % 4]
        both = b[:, 12 + sub % 4]
        sc = torch.where(sub < 4, s & 63, both & 15 | s >> 6 << 4)
        mn = torch.where(sub < 4, t & 63, both >> 4 | t >> 6 << 4)
        out = half(0) * sc * code - half(2) * mn
    else:
        part, quarter, l = i // 128, i % 128 // 32, i % 32
        lo = b[:, 64 * part + 32 * (quarter % 2) + l] >> (4 * (quarter // 2)) & 15
        hi = b[:, 128 + 32 * part + l] >> (2 * quarter) & 3
        out = half(208) * signed(b[:, 192 + i // 16]) * ((lo | hi << 4) - 32)
    return out.reshape(len(w), cols)


def exact(case, seed):
    s = prepare(case, seed)
    op, x = s["op"], s["x"].double()
    if op == "squares":
        if not s["experts"]:
            return {"sums": s["sums"].double() + torch.mm(torch.ones(1, len(x), device="cuda").double(), x.square()),
                    "counts": None}
        sums = s["sums"].double()
        for j in range(s["each"]):
            sums.index_add_(0, s["which"][:, j].long(), x.square())
        return {"sums": sums, "counts": None}
    if op == "project":
        y = torch.mm(x, _weights64(s["w"], s["quant"], s["cols"]).t().contiguous())
        for a in range(s["pool"]):
            at = torch.nonzero(s["which"] == a).reshape(-1)
            low = torch.mm(x[at], s["a"][a].double().t().contiguous())
            y[at] += torch.mm(low, s["b"][a].double().t().contiguous()) * s["scale"][a].double()
        return y
    gate, up = _weights64(s["gate"], s["quant"], s["cols"]), _weights64(s["up"], s["quant"], s["cols"])
    g, u = torch.mm(x, gate.t().contiguous()), torch.mm(x, up.t().contiguous())
    if s["act"] == "silu":
        p = torch.sigmoid(g)
        value, slope = g * p, p + g * p * (1 - p)
    else:                                            # gelu's tanh form as g times a logistic of twice the argument
        c = 2 * math.sqrt(2 / math.pi)
        p = torch.sigmoid(c * g * (1 + 0.044715 * g * g))
        value, slope = g * p, p + g * p * (1 - p) * c * (1 + 0.134145 * g * g)
    if op == "gated":
        return value * u
    dh = s["dh"].double()
    dg, du = dh * u * slope, dh * value
    grads = {"dx": torch.mm(dg, gate).add_(torch.mm(du, up))}
    if s["quant"] in ("F16", "BF16"):
        grads |= {"dgate": torch.mm(dg.t().contiguous(), x), "dup": torch.mm(du.t().contiguous(), x)}
    return grads
