"""Plain 64-bit forms of the dense operators, and how far a result may be off them."""
import math

import numpy as np
import torch

ACTS = ("silu", "gelu", "gelu_tanh", "relu", "sigmoid")


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def tiny(dtype) -> float:
    """Half the distance of the smallest values of a type: what a rounding may be off where values are that small."""
    return float(torch.finfo(dtype).smallest_normal) * half_step(dtype)


def philox(ctr, key):
    """Philox4x32-10: ``ctr`` [..., 4] and ``key`` (2 words) as uint64 arrays of 32-bit values."""
    c = [ctr[..., i].astype(np.uint64) for i in range(4)]
    k = [int(key[0]), int(key[1])]
    m = np.uint64(0xFFFFFFFF)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        s = np.uint64(32)
        c = [(b >> s) ^ c[1] ^ np.uint64(k[0]), b & m, (a >> s) ^ c[3] ^ np.uint64(k[1]), a & m]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, -1)


def drop_factors(rows, cols, p, seed, step=0, row0=0):
    """1 / (1 - p) where an element is kept, 0 where not (float64 tensor)."""
    if p == 0:
        return torch.ones(rows, cols, dtype=torch.float64)
    ctr = np.zeros((rows, (cols + 3) // 4, 4), np.uint64)
    ctr[..., 0] = np.arange(ctr.shape[1])[None, :]
    ctr[..., 1] = (np.arange(rows) + row0)[:, None]
    ctr[..., 2], ctr[..., 3] = step & 0xFFFFFFFF, step >> 32
    w = philox(ctr, (seed & 0xFFFFFFFF, seed >> 32)).reshape(rows, -1)[:, :cols]
    return torch.from_numpy(np.where(w >= np.uint64(int(math.floor(p * 4294967296.0))), 1 / (1 - p), 0.0))


def act(name, g):
    n = torch.nn.functional
    return {"silu": n.silu, "sigmoid": torch.sigmoid, "relu": n.relu, "gelu": n.gelu, "gelu_tanh": lambda v: n.gelu(v, approximate="tanh")}[name](g)


def act_slope(name, g):
    g = g.detach().clone().requires_grad_()
    return torch.autograd.grad(act(name, g).sum(), g)[0]


# FP32 sums of K products (each exact, or rounded to 24 bits): every addition is off by a unit of 2^-23 of the partial sum at most, however it is
# rounded, and the partial sums stay below the sum of the magnitudes.
def sum_bound(K, magnitudes):
    return (K + 2) * 2.0 ** -23 * magnitudes


# The activation in FP32: a handful of roundings and functions good to a few units, absolute in g where a tail cancels (1 + tanh, 1 + erf).
ACT_REL, SLOPE_ABS = 2.0 ** -20, 2.0 ** -18


def gated(x, wg, wu, name, factors, dtype, device="cpu"):
    """h, g, u and the bounds of their errors."""
    x, wg, wu = (t.double().to(device) for t in (x, wg, wu))
    K = x.shape[1]
    g, u = x @ wg, x @ wu
    eg, eu = sum_bound(K, x.abs() @ wg.abs()), sum_bound(K, x.abs() @ wu.abs())
    a = act(name, g)
    h = a * u * factors
    # |act'| <= 1.13 for all of them
    eh = factors * ((1.13 * eg + ACT_REL * (g.abs() + 1)) * (u.abs() + eu) + a.abs() * eu) + 2.0 ** -22 * h.abs()
    hs, t = half_step(dtype), tiny(dtype)
    return (h, g, u), tuple(e + hs * (v.abs() + e) + t for v, e in ((h, eh), (g, eg), (u, eu)))


def gated_grads(dh, x, wg, wu, g, u, name, factors, dtype, device="cpu"):
    """dx, dwg, dwu and the bounds of their errors: dg and du are rounded to the type, then summed in FP32 and rounded again."""
    dh, x, wg, wu, g, u = (t.double().to(device) for t in (dh, x, wg, wu, g, u))
    hs, t = half_step(dtype), tiny(dtype)
    d = dh * factors
    a, s = act(name, g), act_slope(name, g)
    dg, du = d * u * s, d * a
    eg = (d * u).abs() * SLOPE_ABS * (1 + g.abs()) + hs * dg.abs() + t
    eu = d.abs() * ACT_REL * (1 + g.abs()) + hs * du.abs() + t
    F, M = g.shape[1], g.shape[0]

    def out(v, e):
        return v, e + hs * (v.abs() + e) + t

    dx, ex = dg @ wg.T + du @ wu.T, eg @ wg.abs().T + eu @ wu.abs().T
    ex = ex + sum_bound(2 * F, (dg.abs() + eg) @ wg.abs().T + (du.abs() + eu) @ wu.abs().T)
    grads = [out(dx, ex)]
    for v, e in ((dg, eg), (du, eu)):
        grads.append(out(x.T @ v, x.abs().T @ e + sum_bound(M, x.abs().T @ (v.abs() + e))))
    return [v for v, _ in grads], [e for _, e in grads]


def quantize(x):
    """Rows: whole numbers and FP32 scales, by the definition (division in the input's precision, FP32 for 16-bit types)."""
    x = x.cpu()
    w = (x if x.dtype == torch.float64 else x.float()).numpy()
    with np.errstate(all="ignore"):
        most = np.abs(w).max(1) if w.shape[1] else np.zeros(w.shape[0], w.dtype)
        scale = (most / w.dtype.type(127)).astype(np.float32)
        some = (scale > 0) & np.isfinite(scale)
        q = np.clip(np.rint(w / np.where(some, scale, 1).astype(w.dtype)[:, None]), -127, 127)
    return np.where(some[:, None], q, 0).astype(np.int8), scale


def close(got, want, bound, what=""):
    got = got.double().to(want.device)
    assert got.shape == want.shape, what
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got - want).abs() / bound)[bad].max()):.3g} times the bound"
