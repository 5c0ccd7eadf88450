"""The 8-bit integer product and the operators that make its rows, as measured cases.

Ranges.  What a decoder whose matrices are held in 8 bits does between its attention kernels: the norm of the residual
stream with the addition of a sublayer's result, out in 8 bits with a scale for each token; rows brought to 8 bits (the
attention's result, a gated feed-forward's activation); products of such rows with matrices of 8-bit integers and a scale for
each output channel, plain and with a gated activation.  1 to 8192 tokens; widths of 64 to 17408, those of the decoders 1024 to 5120 wide
that ``perf/cases.py`` and ``bench.py`` run among them, and any number beside them: neither tokens nor widths need be multiples of
anything.

The integers come back as they are and have to be equal on both sides: a value's integer is 127 x / max |x| rounded half to even, and both sides
form that quotient in 64 bits.
"""
import math

import torch

#: False: the operators in elementary torch operations; True: the framework's kernels.  The tools set it.
own = False

DEVICE = "cuda:0"
EPS = 1e-6
#: most multiply-adds of a drawn product (those of the largest listed one), and most elements of a drawn norm
MOST_PRODUCT = 4096 * 2 * 12288 * 4096
MOST_ROWS = 8192 * 4096
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def listed():
    return [
        # one user's token through the norm before the attention of an 8B decoder: the launch and the round trip to memory decide
        dict(name="norm/1-token", op="norm", tokens=1, width=4096, addend="bfloat16", weight="bfloat16"),
        # a small batch in a width that is a multiple of nothing, float32 addends and weights
        dict(name="norm/61-odd", op="norm", tokens=61, width=1001, addend="float32", weight="float32"),
        # two full prompts of 4096 tokens in one step
        dict(name="norm/8192", op="norm", tokens=8192, width=4096, addend="bfloat16", weight="bfloat16"),
        # the activation of a feed-forward for eight requests that decode
        dict(name="rows/8-decoding", op="rows", tokens=8, width=12288, dtype="bfloat16"),
        # the same for a prompt, its length a multiple of nothing
        dict(name="rows/2047", op="rows", tokens=2047, width=12288, dtype="bfloat16"),
        # one token's queries, keys and values: the matrix is read once, for one row
        dict(name="product/1-token", op="product", tokens=1, inputs=4096, outputs=6144, out="bfloat16"),
        # the way back from the feed-forward for eight requests: few outputs, a long sum
        dict(name="product/8-decoding", op="product", tokens=8, inputs=12288, outputs=4096, out="bfloat16"),
        # sizes that are multiples of nothing, the sums wanted in float32
        dict(name="product/45-odd", op="product", tokens=45, inputs=1023, outputs=777, out="float32"),
        # a portion of a prompt beside requests that decode: too few tiles for the card, too many rows to stream
        dict(name="product/200", op="product", tokens=200, inputs=4096, outputs=6144, out="bfloat16"),
        # a long prompt
        dict(name="product/4096", op="product", tokens=4096, inputs=12288, outputs=4096, out="bfloat16"),
        # gate and up of a feed-forward with the activation: requests that decode, and a long prompt
        dict(name="gated/16-decoding", op="gated", tokens=16, inputs=4096, outputs=12288, activation="silu"),
        dict(name="gated/4096", op="gated", tokens=4096, inputs=4096, outputs=12288, activation="silu"),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    def width(lo, hi):
        # a decoder's width, a multiple of 64 or 16, or any number
        return rng.choice([rng.choice([w for w in (1024, 2048, 2560, 4096, 5120, 6144, 9728, 12288, 17408) if lo <= w <= hi]),
                           max(1, log(lo, hi) // 64) * 64, max(1, log(lo, hi) // 16) * 16, log(lo, hi)])

    op = rng.choice(["norm", "rows", "product", "product", "gated"])
    if op == "norm":
        w = width(64, 8192)
        return dict(op=op, tokens=min(log(1, 8192), MOST_ROWS // w), width=w, addend=rng.choice(["bfloat16", "bfloat16", "float32", "none"]),
                    weight=rng.choice(["bfloat16", "float32"]))
    if op == "rows":
        w = width(64, 17408)
        return dict(op=op, tokens=min(log(1, 8192), MOST_ROWS // w), width=w, dtype=rng.choice(["bfloat16", "bfloat16", "float32"]))
    if op == "product":
        k, n = width(64, 17408), width(16, 17408)
        return dict(op=op, tokens=min(log(1, 8192), MOST_PRODUCT // (n * k)), inputs=k, outputs=n, out=rng.choice(["bfloat16", "bfloat16", "float32"]))
    k, n = width(64, 8192), width(16, 17408)
    return dict(op=op, tokens=min(log(1, 8192), MOST_PRODUCT // (2 * n * k)), inputs=k, outputs=n, activation=rng.choice(["silu", "silu", "gelu_tanh"]))


def _activations(shape, g):
    """Activations as a decoder has them: every row has a size of its own, and one channel in 50 is ten times the others."""
    x = torch.randn(shape, device=DEVICE, generator=g)
    x *= torch.exp(0.5 * torch.randn((shape[0], 1), device=DEVICE, generator=g))
    x *= torch.where(torch.rand((1, shape[1]), device=DEVICE, generator=g) < 0.02, 10.0, 1.0)
    return x


def _integers(x):
    """(int8 values, float32 scales) of rows: what a checkpoint in 8 bits, or the operator before, has left."""
    a = x.abs().amax(dim=1, keepdim=True).clamp_min(1e-20)
    return torch.round(x * (127.0 / a)).clamp_(-127, 127).to(torch.int8), (a / 127.0).reshape(-1)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    s = dict(op=case["op"])
    if case["op"] == "norm":
        shape = (case["tokens"], case["width"])
        s["stream"] = _activations(shape, g)
        s["addend"] = None if case["addend"] == "none" else (0.3 * _activations(shape, g)).to(DTYPES[case["addend"]])
        s["weight"] = (1.0 + 0.2 * torch.randn((case["width"],), device=DEVICE, generator=g)).to(DTYPES[case["weight"]])
        return s
    if case["op"] == "rows":
        s["x"] = _activations((case["tokens"], case["width"]), g).to(DTYPES[case["dtype"]])
        return s
    gated = case["op"] == "gated"
    n, k = case["outputs"] * (2 if gated else 1), case["inputs"]
    x, sx = _integers(_activations((case["tokens"], k), g))
    w, sw = _integers(torch.randn((n, k), device=DEVICE, generator=g) / math.sqrt(k))
    s.update(tokens=case["tokens"], activation=case.get("activation"), out=DTYPES[case.get("out", "bfloat16")])
    if own:
        from spyinfer_amd.kernels import ops
        # the rows as the operator before leaves them, the matrix laid out as a model keeps it
        s["rows"], s["matrix"] = ops.Q8Rows.from_values(x, sx), ops.Q8Weight.from_values(w, sw, gated=gated)
    else:
        s.update(x=x, sx=sx, w=w, sw=sw)
    return s


def run(s):
    if own:
        from spyinfer_amd.kernels import ops
        if s["op"] == "norm":
            rows = ops.add_rms_norm_q8(s["stream"], s["addend"], s["weight"], EPS)
            return {"stream": s["stream"], "values": rows.values[:, :rows.width], "scales": rows.scales}
        if s["op"] == "rows":
            rows = ops.quantize_rows(s["x"])
            return {"values": rows.values[:, :rows.width], "scales": rows.scales}
        if s["op"] == "product":
            return ops.linear_q8(s["rows"], s["matrix"], s["out"])
        return ops.linear_q8_gated(s["rows"], s["matrix"], s["activation"])
    if s["op"] == "norm":
        x = s["stream"]
        if s["addend"] is not None:
            x.add_(s["addend"].float())
        rms = torch.sqrt(torch.mean(x * x, dim=1) + EPS)
        z = x.double() * s["weight"].double()
        top = z.abs().amax(dim=1)
        # (a value next to the border of two integers needs the quotient in 64 bits; the norm's factor does not enter it)
        return {"stream": x, "values": _rounded(z, top), "scales": (top / 127.0 / rms.double()).float()}
    if s["op"] == "rows":
        x = s["x"].double()
        top = x.abs().amax(dim=1)
        return {"values": _rounded(x, top), "scales": (top / 127.0).float()}
    y = torch.matmul(s["x"].float(), s["w"].float().t()) * s["sx"][:, None] * s["sw"][None, :]
    if s["op"] == "product":
        return y.to(s["out"])
    gate, up = y.chunk(2, dim=1)
    return (_activation(gate, s["activation"]) * up).to(torch.bfloat16)


def _rounded(z, top):
    return torch.round(z * 127.0 / torch.where(top > 0, top, 1.0)[:, None]).to(torch.int8)


def _activation(z, name):
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))


def work(case):
    size = {"bfloat16": 2, "float32": 4, "none": 0}
    t = case["tokens"]
    if case["op"] == "norm":
        h = case["width"]
        return {"bytes": t * h * (4 + size[case["addend"]] + 4 + 1) + h * size[case["weight"]] + 4 * t, "flops": 8 * t * h}
    if case["op"] == "rows":
        return {"bytes": t * case["width"] * (size[case["dtype"]] + 1) + 4 * t, "flops": 3 * t * case["width"]}
    n, k = case["outputs"], case["inputs"]
    m = 2 * n if case["op"] == "gated" else n
    return {"bytes": t * k + m * k + 4 * (t + m) + t * n * size[case.get("out", "bfloat16")], "flops": 2 * t * m * k}


def exact(case, seed):
    """From the definitions in 64 bits, a sum of integers as a product of float64, which holds it exactly."""
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "norm":
        stream = s["stream"].double() if s["addend"] is None else (s["stream"] + s["addend"].float()).double()
        normed = stream / torch.sqrt((stream ** 2).sum(dim=1, keepdim=True) / case["width"] + EPS) * s["weight"].double()
        top = torch.max(normed.abs(), dim=1).values
        return {"stream": stream, "values": torch.round(normed * 127.0 / top[:, None]).to(torch.int8), "scales": top / 127.0}
    if case["op"] == "rows":
        x = s["x"].double()
        top = torch.max(x.abs(), dim=1).values
        return {"values": torch.round(x * 127.0 / top[:, None]).to(torch.int8), "scales": top / 127.0}
    q = s["x"].double() * s["sx"].double().reshape(-1, 1)
    p = s["w"].double() * s["sw"].double().reshape(-1, 1)
    y = q @ p.transpose(0, 1)
    if case["op"] == "product":
        return y
    half = case["outputs"]
    z, up = y[:, :half], y[:, half:]
    if case["activation"] == "silu":
        return z * torch.sigmoid(z) * up
    # z/2 (1 + tanh(u)) = z sigmoid(2 u)
    return z * torch.sigmoid(2.0 * (2.0 / math.pi) ** 0.5 * (z + 0.044715 * z ** 3)) * up
