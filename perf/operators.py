"""Performance cases of the dense operators beside the compressed products, as a program that uses this package calls them.

* ``op`` "q8"       out = (x in 8 bits) %*% (weights in 8 bits), a scale per row of x and per column of the weights. ``dynamic``: x comes
                    in ``dtype`` and is quantised in the pass, as activations are; else it is in 8 bits already
* ``op`` "forward"  H = act(X Wg) * (X Wu), the gated block, with dropout of H where ``p`` > 0; ``save``: X Wg and X Wu come out too
* ``op`` "backward" dX, dWg, dWu of it from dH and the saved X Wg, X Wu
* ``op`` "dropout"  y = x * keep / (1 - p), keep from a counter-based generator (Philox4x32-10, Salmon et al. 2011)

``rows`` of x, ``inner`` its columns, ``cols`` the weights' columns; ``packed``: both weights lie side by side in one matrix (their rows
are then twice as far apart as they are long), for "q8" and "dropout" x is a part of wider rows.

Where ``own`` is false the operators are computed in elementary torch operations. ``exact`` computes them in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _case(name, op, rows, inner, cols, dtype="bf16", act="", p=0.0, save=False, packed=False, dynamic=False):
    c = {"op": op, "rows": rows, "inner": inner, "cols": cols, "dtype": dtype, "act": act, "p": p, "save": save, "packed": packed,
         "dynamic": dynamic}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one token through a layer served in 8 bits: latency, and the weights read once
        _case("q8_token", "q8", 1, 4096, 8192, dynamic=True),
        # a few requests decoded together, a column count that no tile divides
        _case("q8_few", "q8", 24, 2048, 10007, "fp16", dynamic=True),
        # class scores of a decompressed block of odd width, 64 classes, in the precision that the block's products have
        _case("q8_scores", "q8", 100_003, 501, 64, "f64", dynamic=True),
        # a batch of prompts, activations quantised by the layer before
        _case("q8_batch", "q8", 8192, 4096, 16384),
        # one token through the hidden layer: latency, and both weights read once
        _case("gate_token", "forward", 1, 4096, 16384, act="silu"),
        # a few requests decoded together, weights side by side in one matrix
        _case("gate_few", "forward", 40, 2048, 5504, "fp16", act="gelu_tanh", packed=True),
        # a training step's forward half with dropout, odd row count and a hidden width that no 16-byte row holds
        _case("gate_train_odd", "forward", 4095, 2048, 5461, "fp16", act="gelu", p=0.1, save=True),
        # a batch of prompts
        _case("gate_batch", "forward", 8192, 4096, 12288, act="silu"),
        # a training step's backward half with dropout
        _case("gate_back", "backward", 8192, 2048, 8192, act="silu", p=0.1),
        # the same with few odd rows and odd widths
        _case("gate_back_odd", "backward", 777, 1001, 2731, "fp16", act="gelu"),
        # activations of one block of rows
        _case("dropout_block", "dropout", 1000, 0, 100, "f32", p=0.5),
        # hidden activations of a batch
        _case("dropout_batch", "dropout", 16384, 0, 8192, p=0.1),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the listed ranges: sizes log-uniform, every other one rounded to a multiple of 8, never more work than the largest listed
    case of its operator."""
    op = rng.choice(["q8", "q8", "forward", "forward", "backward", "backward", "dropout"])
    even = rng.random() < 0.5
    size = lambda lo, hi: max(8, _log(rng, lo, hi) // 8 * 8) if even else _log(rng, lo, hi)  # noqa: E731
    packed = rng.random() < 0.3
    if op == "dropout":
        rows, cols = _log(rng, 1, 16384), size(64, 8192)
        return _case(None, op, rows, 0, cols, rng.choice(["f64", "f32", "bf16", "fp16"]), p=rng.choice([0.1, 0.25, 0.5]), packed=packed)
    if op == "q8":
        rows, inner, cols = _log(rng, 1, 8192), size(100, 8192), size(64, 16384)
        rows = max(1, min(rows, int(5.4e11 / inner / cols)))
        dynamic = rng.random() < 0.7
        return _case(None, op, rows, inner, cols, rng.choice(["f64", "f32", "bf16", "bf16", "fp16"]), packed=packed, dynamic=dynamic)
    rows, inner, cols = _log(rng, 1, 8192), size(100, 4096), size(100, 16384)
    rows = max(1, min(rows, int((4e11 if op == "forward" else 1.3e11) / inner / cols)))
    act = rng.choice(["silu", "gelu", "gelu_tanh", "relu", "sigmoid"])
    return _case(None, op, rows, inner, cols, rng.choice(["bf16", "fp16"]), act, rng.choice([0.0, 0.1]), op == "forward" and rng.random() < 0.5,
                 packed)


# ---- inputs -------------------------------------------------------------------------------------------------------
def _normal(gen, rows, cols, dtype, scale=1.0, wide=False):
    """Normal values; `wide`: as the middle part of longer rows."""
    pad = cols + 24 if wide else cols
    x = (torch.randn(rows, pad, device="cuda", generator=gen) * scale).to(dtype)
    return x[:, 16:16 + cols] if wide else x


def _in_8_bits(x):
    """Rows of x as whole numbers in -127..127 and their scales: fl32(largest magnitude / 127), x / scale to the nearest, even on ties."""
    wide = x.double() if x.dtype == torch.float64 else x.float()
    scale = (wide.abs().amax(1) / 127).float()
    q = torch.round(wide / scale.to(wide.dtype)[:, None]).clamp(-127, 127)
    q = torch.where((scale > 0) & torch.isfinite(scale), q.T, 0).T
    return q.to(torch.int8), scale


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 1_000_003 + 29)
    t = DTYPES[c["dtype"]]
    rows, inner, cols = c["rows"], c["inner"], c["cols"]
    c["seed"], c["step"] = seed * 7919 + 13, seed % 97
    if c["op"] == "dropout":
        c["x"] = _normal(gen, rows, cols, t, wide=c["packed"])
        return c
    x = _normal(gen, rows, inner, t, wide=c["packed"] and c["op"] == "q8")
    if c["op"] == "q8":
        # weights as a program keeps them: quantised once, a row per output column
        c["b"], c["bScale"] = _in_8_bits(_normal(gen, cols, inner, torch.float32, inner ** -0.5))
        if c["dynamic"]:
            c["x"] = x
        else:
            c["a"], c["aScale"] = _in_8_bits(x)
        return c
    c["x"] = x
    if c["packed"]:
        w = _normal(gen, inner, 2 * cols, t, inner ** -0.5)
        c["wg"], c["wu"] = w[:, :cols], w[:, cols:]
    else:
        c["wg"], c["wu"] = _normal(gen, inner, cols, t, inner ** -0.5), _normal(gen, inner, cols, t, inner ** -0.5)
    if c["op"] == "backward":  # what the forward half has saved
        c["g"], c["u"] = x @ c["wg"], x @ c["wu"]
        c["dh"] = _normal(gen, rows, cols, t)
    return c


# ---- plain forms ---------------------------------------------------------------------------------------------------
_M = 0xFFFFFFFF


def _words(rows, cols, seed, step):
    """Philox4x32-10 with key `seed` and counter (column / 4, row, step): the words of a [rows x cols] tensor, as 64-bit integers."""
    n = (cols + 3) // 4
    c0 = torch.arange(n, device="cuda")[None, :].expand(rows, n)
    c1 = torch.arange(rows, device="cuda")[:, None].expand(rows, n)
    c2, c3 = torch.full_like(c0, step & _M), torch.full_like(c0, step >> 32)
    k0, k1 = seed & _M, seed >> 32
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # (wrapped products keep the bits)
        c0, c1, c2, c3 = ((b >> 32) & _M) ^ c1 ^ k0, b & _M, ((a >> 32) & _M) ^ c3 ^ k1, a & _M
        k0, k1 = (k0 + 0x9E3779B9) & _M, (k1 + 0xBB67AE85) & _M
    return torch.stack([c0, c1, c2, c3], 2).reshape(rows, 4 * n)[:, :cols]


def _kept(x, c):
    """x with the dropped values at zero and the others scaled."""
    if c["p"] == 0:
        return x
    keep = _words(x.shape[0], x.shape[1], c["seed"], c["step"]) >= int(c["p"] * 2.0 ** 32)
    return torch.where(keep, x * (1 / (1 - c["p"])), 0)


def _act(name, g):
    if name == "silu":
        return g / (1 + torch.exp(-g))
    if name == "sigmoid":
        return 1 / (1 + torch.exp(-g))
    if name == "relu":
        return torch.clamp(g, min=0)
    if name == "gelu":
        return 0.5 * g * (1 + torch.erf(g * 0.5 ** 0.5))
    return 0.5 * g * (1 + torch.tanh((2 / math.pi) ** 0.5 * (g + 0.044715 * g * g * g)))


def _act_slope(name, g):
    if name == "silu":
        s = 1 / (1 + torch.exp(-g))
        return s * (1 + g * (1 - s))
    if name == "sigmoid":
        s = 1 / (1 + torch.exp(-g))
        return s * (1 - s)
    if name == "relu":
        return (g > 0).to(g.dtype)
    if name == "gelu":
        return 0.5 * (1 + torch.erf(g * 0.5 ** 0.5)) + g * torch.exp(-0.5 * g * g) * (2 * math.pi) ** -0.5
    k = (2 / math.pi) ** 0.5
    t = torch.tanh(k * (g + 0.044715 * g * g * g))
    return 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * k * (1 + 3 * 0.044715 * g * g)


def _plain(c):
    t = DTYPES[c["dtype"]]
    if c["op"] == "dropout":
        return _kept(c["x"].double() if t == torch.float64 else c["x"].float(), c).to(t)
    if c["op"] == "q8":
        a, scale = _in_8_bits(c["x"]) if c["dynamic"] else (c["a"], c["aScale"])
        # sums beyond 2^24: in 64 bits
        return ((a.double() @ c["b"].double().T) * scale.double()[:, None] * c["bScale"].double()).to(t)
    x, wg, wu = c["x"].float(), c["wg"].float(), c["wu"].float()
    if c["op"] == "forward":
        g, u = x @ wg, x @ wu
        h = _kept(_act(c["act"], g) * u, c).to(t)
        return (h, g.to(t), u.to(t)) if c["save"] else h
    g, u, dh = c["g"].float(), c["u"].float(), _kept(c["dh"].float(), c)
    dg, du = dh * u * _act_slope(c["act"], g), dh * _act(c["act"], g)
    return (dg @ wg.T + du @ wu.T).to(t), (x.T @ dg).to(t), (x.T @ du).to(t)


def run(c):
    if not own:
        return _plain(c)
    from systemds_b200 import CLALibDropout, CLALibGated, CLALibQ8
    if c["op"] == "dropout":
        return CLALibDropout.apply(c["x"], c["p"], c["seed"], c["step"])
    if c["op"] == "q8":
        if c["dynamic"]:
            return CLALibQ8.linear(c["x"], c["b"], c["bScale"])
        return CLALibQ8.matrixMult(c["a"], c["aScale"], c["b"], c["bScale"], DTYPES[c["dtype"]])
    if c["op"] == "forward":
        return CLALibGated.forward(c["x"], c["wg"], c["wu"], c["act"], p=c["p"], seed=c["seed"], step=c["step"], save=c["save"])
    return CLALibGated.backward(c["dh"], c["x"], c["wg"], c["wu"], c["g"], c["u"], c["act"], p=c["p"], seed=c["seed"], step=c["step"])


def work(case):
    m, k, n, b = case["rows"], case["inner"], case["cols"], torch.finfo(DTYPES[case["dtype"]]).bits // 8
    if case["op"] == "dropout":
        return {"bytes": 2 * m * n * b, "flops": m * n}
    if case["op"] == "q8":
        return {"bytes": m * k * (b if case["dynamic"] else 1) + n * k + 4 * n + (0 if case["dynamic"] else 4 * m) + m * n * b, "flops": 2 * m * n * k}
    if case["op"] == "forward":
        return {"bytes": b * (m * k + 2 * k * n + m * n * (3 if case["save"] else 1)), "flops": 4 * m * n * k}
    return {"bytes": b * (3 * m * n + 2 * m * k + 4 * k * n), "flops": 8 * m * n * k}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------
def _times(a, m):
    """High and low 32 bits of a * m, from products of 16-bit halves."""
    lo, hi = a & 0xFFFF, a >> 16
    x, y = lo * (m & 0xFFFF), lo * (m >> 16)
    z, w = hi * (m & 0xFFFF), hi * (m >> 16)
    mid = (x >> 16) + (y & 0xFFFF) + (z & 0xFFFF)
    return (w + (y >> 16) + (z >> 16) + (mid >> 16)) & _M, ((mid & 0xFFFF) << 16) | (x & 0xFFFF)


def _factors(c):
    """1 / (1 - p) or 0 for every value, row block by row block."""
    rows, cols, cut = c["rows"], c["cols"], math.floor(c["p"] * 4294967296.0)
    out = torch.ones(rows, cols, dtype=torch.float64, device="cuda")
    if c["p"] == 0:
        return out
    for r0 in range(0, rows, 2048):
        n = min(2048, rows - r0)
        col = torch.arange(cols, device="cuda").repeat(n, 1)
        v = [col // 4, torch.arange(r0, r0 + n, device="cuda")[:, None].expand(n, cols), torch.full_like(col, c["step"] % 2 ** 32),
             torch.full_like(col, c["step"] // 2 ** 32)]
        key = [c["seed"] % 2 ** 32, c["seed"] // 2 ** 32]
        for _ in range(10):
            h0, l0 = _times(v[0], 0xD2511F53)
            h1, l1 = _times(v[2], 0xCD9E8D57)
            v = [h1 ^ v[1] ^ key[0], l1, h0 ^ v[3] ^ key[1], l0]
            key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
        word = torch.gather(torch.stack(v), 0, (col % 4)[None])[0]
        out[r0:r0 + n] = (word >= cut).double() / (1 - c["p"])
    return out


def _act_exact(name, g):
    n = torch.nn.functional
    return {"silu": n.silu, "sigmoid": torch.sigmoid, "relu": n.relu, "gelu": n.gelu, "gelu_tanh": lambda v: n.gelu(v, approximate="tanh")}[name](g)


def exact(case, seed):
    c = prepare(case, seed)
    if c["op"] == "dropout":
        return c["x"].double() * _factors(c)
    if c["op"] == "q8":
        a, scale = _in_8_bits(c["x"]) if c["dynamic"] else (c["a"], c["aScale"])
        a, b = a.double() * scale.double().unsqueeze(1), c["b"].double() * c["bScale"].double().unsqueeze(1)
        return torch.cat([part @ b.T for part in a.split(4096)])
    x, wg, wu = c["x"].double(), c["wg"].double(), c["wu"].double()
    if c["op"] == "forward":
        g, u = torch.mm(x, wg), torch.mm(x, wu)
        h = _act_exact(c["act"], g) * u * _factors(c)
        return (h, g, u) if c["save"] else h
    g, u = c["g"].double().requires_grad_(), c["u"].double().requires_grad_()
    dg, du = torch.autograd.grad(_act_exact(c["act"], g) * u, (g, u), c["dh"].double() * _factors(c))
    both = torch.cat([dg, du], 1)
    dw = x.T @ both
    n = c["cols"]
    return both @ torch.cat([wg, wu], 1).T, dw[:, :n], dw[:, n:]
