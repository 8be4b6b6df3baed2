"""The dense operators on the GPU where a tail, another caller or an odd argument shows what the bounds of test_dense_gpu.py do not."""
import math
import os
import subprocess
import sys

import pytest
import torch

from systemds_b200 import CLAError, CLALibDecompress, CLALibDropout, CLALibGated, CLALibQ8, datagen, native
from systemds_b200.dense import status
from tests import dense_ref as ref

pytestmark = pytest.mark.gpu
HALVES = (torch.bfloat16, torch.float16)


@pytest.fixture(autouse=True)
def no_check_trips():
    yield
    status()


# ---- activations in their tails -----------------------------------------------------------------------------------------
def gates_of(dtype, most):
    """Every value of a 16-bit type from 2^-6 to `most` in magnitude, and zero."""
    v = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(dtype)
    m = v.double().abs()
    return torch.cat([v[(m >= 2.0 ** -6) & (m <= most)], torch.zeros(1, dtype=dtype)])


def tail_forms(act, g):
    """act(g), act'(g) without a cancelling sum, and the magnitudes that its relative error counts from (their sum may pass through zero), both with the
    error of a float32 evaluation in units of 2^-23: a documented 2 + 1.173 |x| for the exponential of x, 2 for the quotient, what a rounding of the
    argument x is worth, |x| / 2 each, 1/2 for each other rounding, and 4.4 for a polynomial of degree 8 in GELU's tail (2 + 1.173 g^2 / 2 + g^2 / 2 + 4.4 + 1 for that)."""
    s, r = torch.sigmoid(g), torch.sigmoid(-g)
    a = g.abs()
    if act == "relu":
        return g.clamp(min=0), (g > 0).double(), (g > 0).double(), 0 * a, 0 * a
    if act == "sigmoid":
        return s, s * r, s * r, 6 + 1.2 * a, 20 + 3.6 * a
    if act == "silu":
        return g * s, s + g * s * r, s + a * s * r, 6 + 1.2 * a, 20 + 3.6 * a
    if act == "gelu":
        c = 0.5 * torch.special.erfc(-g / math.sqrt(2))
        p = g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
        return g * c, c + p, c + p.abs(), 10 + 1.2 * g * g, 12 + 1.2 * g * g
    k = math.sqrt(8 / math.pi)  # (1 + tanh(y)) / 2 = sigmoid(2 y)
    y = k * (g + 0.044715 * g ** 3)
    s, r, d = torch.sigmoid(y), torch.sigmoid(-y), k * (1 + 3 * 0.044715 * g * g)
    return g * s, s + g * s * r * d, s + a * s * r * d, 6 + 3.2 * y.abs(), 20 + 9.6 * y.abs()


@pytest.mark.parametrize("rows", [1, 300])
@pytest.mark.parametrize("dtype,most,scale", [(torch.bfloat16, 110.0, 1.0), (torch.float16, 20.0, 512.0)])
@pytest.mark.parametrize("act", ref.ACTS)
def test_activations_hold_their_relative_error_in_the_tails(act, dtype, most, scale, rows):
    """One column of ones times the gates: the products are the gates themselves, and the weights' gradients dG and dU of a single row."""
    gate = gates_of(dtype, most).cuda()
    F, g = len(gate), gate.double().cpu()
    up = torch.full((1, F), scale, dtype=dtype, device="cuda")
    x = torch.ones((rows, 1), dtype=dtype, device="cuda")
    value, slope, mags, ulps, slope_ulps = tail_forms(act, g)
    half, tiny, unit = ref.half_step(dtype), ref.tiny(dtype), 2.0 ** -23

    def holds(got, want, ulps, mags, what):
        # (the float32 error, the scaling's rounding, then the type's; below 2^-126 float32 has steps of 2^-149)
        e = scale * mags.abs() * (ulps + 2) * unit + scale * (1 + g.abs()) * 2.0 ** -147
        ref.close(got, want * scale, e + half * ((want * scale).abs() + e) + tiny, what)

    h = CLALibGated.forward(x, gate[None], up, act)
    assert torch.equal(h, h[:1].expand_as(h))
    holds(h[0], value, ulps, value, "value")
    if rows == 1:
        one = torch.ones((1, F), dtype=dtype, device="cuda")
        _, dwg, dwu = CLALibGated.backward(up, x, gate[None], one, gate[None], one, act, needX=False)
        holds(dwg[0], slope, slope_ulps, mags, "slope")
        holds(dwu[0], value, ulps, value, "value in the gradient")


# ---- results next to operands -------------------------------------------------------------------------------------------
def test_results_onto_operands_are_refused():
    """Shapes that fit: it is the shared memory that refuses the call, and nothing has been written."""
    x = torch.randn(40, 64, device="cuda").to(torch.bfloat16)
    w = torch.randn(64, 64, device="cuda").to(torch.bfloat16)
    keep, keepW = x.clone(), w.clone()
    q, s = CLALibQ8.quantizeCols(w)
    for f in (lambda: CLALibGated.forward(x, w, w, out=x), lambda: CLALibGated.forward(w, w, keepW, out=w), lambda: CLALibQ8.linear(x, q, s, out=x),
              lambda: CLALibDropout.apply(x[:39], 0.5, 1, out=x[1:])):
        with pytest.raises(CLAError):
            f()
    assert torch.equal(x, keep) and torch.equal(w, keepW)


def test_results_beside_operands_in_the_same_rows_are_taken():
    w = torch.randn(64, 64, device="cuda").to(torch.bfloat16)
    q, s = CLALibQ8.quantizeCols(w)
    wide = torch.randn(50, 200, device="cuda").to(torch.bfloat16)
    x, out = wide[:, 3:67], wide[:, 67:131]
    want = CLALibGated.forward(x.clone(), w, w), CLALibQ8.linear(x.clone(), q, s), CLALibDropout.apply(x.clone(), 0.5, 1)
    for f, v in zip((lambda: CLALibGated.forward(x, w, w, out=out), lambda: CLALibQ8.linear(x, q, s, out=out),
                     lambda: CLALibDropout.apply(x, 0.5, 1, out=out)), want):
        assert torch.equal(f(), v) and torch.equal(out, v)
    x, out = wide[:25, 3:67], wide.view(25, 400)[:, 270:334]  # rows twice as far apart as the operand's
    want = CLALibDropout.apply(x.clone(), 0.5, 1)
    assert torch.equal(CLALibDropout.apply(x, 0.5, 1, out=out), want)
    with pytest.raises(CLAError):
        CLALibDropout.apply(x, 0.5, 1, out=wide.view(25, 400)[:, 266:330])


# ---- a compressed block's calls, captured -------------------------------------------------------------------------------
@pytest.mark.parametrize("rows", [3000, 700_000])  # (the larger one in chunks, the second of which finds a plan worth building)
def test_block_calls_captured_between_direct_ones(rows):
    """Direct calls on the default stream, captured ones on another, replays, and direct calls on a third stream and again on the first."""
    cmb = datagen.random_cmb(3, rows, datagen.KINDS).to_device(0)
    w, scale = CLALibQ8.quantizeCols(torch.randn(cmb.clen, 33, device="cuda"))
    V = torch.randn(cmb.clen, 2, device="cuda", dtype=torch.float64)

    def calls():
        product = torch.empty((rows, 2), device="cuda", dtype=torch.float64)
        native.check(native.lib().cla_rmm_dev(cmb.handle(), V.data_ptr(), cmb.clen, 2, product.data_ptr(), torch.cuda.current_stream().cuda_stream))
        return CLALibDecompress.rows(cmb, 5, rows - 7, torch.float32), CLALibQ8.rightMultByMatrix(cmb, w, scale), product

    def same(got):
        torch.cuda.synchronize()
        return all(torch.equal(p, q) for p, q in zip(got, want))

    want = calls()
    torch.cuda.synchronize()
    side, other, third = torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.Stream()
    graphs = []
    for fork in (False, True):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = calls()
            if fork:  # the handle's calls on two streams of one capture
                other.wait_stream(side)
                with torch.cuda.stream(other):
                    out += calls()
                side.wait_stream(other)
                out += calls()
        graphs.append((graph, out))
        assert same(calls())
    for graph, out in graphs * 2:
        for t in out:
            t.zero_()
        graph.replay()
        assert same(out[:3]) and same(out[-3:]) and same(out[len(out) // 3:][:3] if len(out) > 3 else out)
        with torch.cuda.stream(third):
            got = calls()
        assert same(got) and same(calls())
    del graphs, graph
    cmb.free()


def test_rows_of_a_block_whose_end_leaves_64_bits():
    cmb = datagen.random_cmb(3, 3000, datagen.KINDS).to_device(0)
    L, h = native.lib(), cmb.handle()
    out = torch.full((8, cmb.clen), 7.0, device="cuda")
    n = native.check(L.cla_rows_workspace(h, 8, 1))
    work = torch.empty(n, dtype=torch.uint8, device="cuda")
    for row0, rows in (((1 << 63) - 1, 8), ((1 << 63) - 8, 8), (2993, 8), (-1, 8), (0, (1 << 63) - 1), (1, (1 << 63) - 1)):
        with pytest.raises(CLAError) as e:
            native.check(L.cla_decompress_rows_dev(h, row0, rows, 1, out.data_ptr(), cmb.clen, work.data_ptr(), n, None))
        assert e.value.code == -4
    for N in (1 << 31, 1 << 56, (1 << 63) - 1):
        with pytest.raises(CLAError) as e:
            native.check(L.cla_q8_rmm_workspace(h, N))
        assert e.value.code == -3
    assert bool((out == 7).all())
    cmb.free()


def test_arguments_of_other_kinds_on_the_device():
    x = torch.ones((8, 16), device="cuda", dtype=torch.bfloat16)
    w, q, s = x.t().contiguous(), *CLALibQ8.quantizeRows(x)
    for f in (lambda: CLALibQ8.linear(x, q, s, dtype="bf16"), lambda: CLALibQ8.linear(x, q, s, dtype=0), lambda: CLALibQ8.matrixMult(q, s, q, s, None),
              lambda: CLALibGated.forward(x, w, w, ["silu"]), lambda: CLALibGated.forward(x, w, w, p="0.1"), lambda: CLALibGated.forward(x, w, w, seed=0.5),
              lambda: CLALibDropout.apply(x, None, 1), lambda: CLALibQ8.linear(x, [q], s), lambda: CLALibQ8.linear(x, q, [s])):
        with pytest.raises(CLAError):
            f()
    seed = torch.tensor(5)
    assert torch.equal(CLALibDropout.apply(x, torch.tensor(0.5), seed), CLALibDropout.apply(x, 0.5, 5))


# ---- several host threads -----------------------------------------------------------------------------------------------
THREADS = """
import threading, torch
from systemds_b200 import CLALibDropout, CLALibGated, CLALibQ8
from systemds_b200.dense import status
torch.cuda.init()
inputs = []
for i, (M, D, F) in enumerate([(1, 512, 900), (40, 300, 700), (700, 264, 333), (2000, 128, 512), (300, 64, 2500), (3000, 200, 64)]):
    g = torch.Generator(device="cuda")
    g.manual_seed(i)
    make = lambda *s: torch.randn(*s, device="cuda", generator=g).half()
    inputs.append((make(M, D), make(D, F) / 16, make(D, F) / 16, make(M, F), torch.randint(-127, 128, (F, D), dtype=torch.int8, device="cuda", generator=g),
                   torch.rand(F, device="cuda", generator=g)))
torch.cuda.synchronize()

def work(k):
    x, wg, wu, dh, b, s = inputs[k % len(inputs)]
    h, g, u = CLALibGated.forward(x, wg, wu, "gelu", p=0.1, seed=3, save=True)
    return (h, CLALibQ8.linear(x, b, s), CLALibDropout.apply(x, 0.5, 7)) + CLALibQ8.quantizeCols(wg) + CLALibGated.backward(dh, x, wg, wu, g, u, "gelu", p=0.1, seed=3)

got, start = {}, threading.Barrier(8)

def run(t):
    stream = torch.cuda.Stream()
    start.wait()
    with torch.cuda.stream(stream):
        for turn in range(12):
            got[t, turn] = work(t + turn)
    stream.synchronize()

threads = [threading.Thread(target=run, args=(t,)) for t in range(8)]
[t.start() for t in threads]
[t.join() for t in threads]
torch.cuda.synchronize()
want = [work(k) for k in range(len(inputs))]
assert len(got) == 96
for (t, turn), r in got.items():
    assert all(torch.equal(p, q) for p, q in zip(r, want[(t + turn) % len(inputs)])), (t, turn)
status()
print("ok")
"""


def test_first_calls_of_several_threads():
    """Eight host threads whose first calls in the process meet, a stream each: the results of calls one after another."""
    r = subprocess.run([sys.executable, "-c", THREADS], capture_output=True, text=True, timeout=300,
                       cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr
