"""The dense operators on the GPU against their plain 64-bit forms (tests/dense_ref.py, where the bounds are derived)."""
import ctypes as C

import numpy as np
import pytest
import torch

from systemds_b200 import CLAError, CLALibDecompress, CLALibDropout, CLALibGated, CLALibQ8, datagen, native
from systemds_b200.dense import status
from tests import dense_ref as ref
from tests.util import dense_of

pytestmark = pytest.mark.gpu
HALVES = (torch.bfloat16, torch.float16)
FLOATS = (torch.float64, torch.float32) + HALVES


@pytest.fixture(autouse=True)
def no_check_trips():
    yield
    status()


def normal(rows, cols, dtype, seed, scale=1.0, pad=0):
    """Normal values; ``pad``: inside a larger matrix of NaN, rows ``cols + pad`` apart, so that nothing around them may reach a result."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    v = (torch.randn(rows, cols, device="cuda", generator=gen, dtype=torch.float64) * scale).to(dtype)
    if not pad:
        return v
    wide = torch.full((rows + 2, cols + pad), float("nan"), device="cuda", dtype=dtype)
    part = wide[1:rows + 1, pad // 2:pad // 2 + cols]
    part.copy_(v)
    return part


def framed(rows, cols, dtype):
    """A result inside a larger matrix of 7, and whether what is around it still is 7."""
    wide = torch.full((rows + 2, cols + 5), 7.0, device="cuda").to(dtype)
    part = wide[1:rows + 1, 3:3 + cols]

    def intact():
        w = wide.clone()
        w[1:rows + 1, 3:3 + cols] = 7
        return bool((w == 7).all())

    return part, intact


# ---- dropout --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows,cols,pad", [(1, 1, 0), (3, 5, 0), (64, 1000, 0), (257, 1023, 0), (40, 96, 16), (33, 41, 7)])
def test_dropout(dtype, rows, cols, pad):
    x = normal(rows, cols, dtype, rows + cols, pad=pad)
    for p, seed, step, row0 in ((0.0, 1, 0, 0), (0.3, 5, 7, 0), (0.5, (1 << 64) - 3, (1 << 40) + 1, (1 << 32) - rows)):
        y, intact = framed(rows, cols, dtype)
        CLALibDropout.apply(x, p, seed, step, row0, out=y)
        f = ref.drop_factors(rows, cols, p, seed, step, row0)
        want = x.double().cpu() * f
        assert torch.equal(y.cpu() == 0, (f == 0) | (want == 0))
        # the factor rounded to FP32 (FP64 for FP64), the product to FP32 and to the type
        ref.close(y, want, want.abs() * (2.0 ** -52 if dtype == torch.float64 else ref.half_step(dtype) + 2.0 ** -22) + ref.tiny(dtype))
        assert intact()


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows,cols", [(7, 1101), (9, 301), (4, 259), (40, 5003), (1300, 257)])
def test_dropout_of_rows_that_start_anywhere(dtype, rows, cols):
    """Rows at every offset from a 16-byte boundary, into other rows at other offsets and onto themselves."""
    f = ref.drop_factors(rows, cols, 0.25, 11, 3)
    for start, ld in ((1, cols), (2, cols + 2), (3, cols + 5)):
        flat = torch.full((start + rows * ld + 8,), float("nan"), device="cuda", dtype=dtype)
        x = flat[start:start + rows * ld].view(rows, ld)[:, :cols]
        x.copy_(normal(rows, cols, dtype, start))
        keep = x.clone()
        want = keep.double().cpu() * f
        bound = want.abs() * (2.0 ** -52 if dtype == torch.float64 else ref.half_step(dtype) + 2.0 ** -22) + ref.tiny(dtype)
        y, intact = framed(rows, cols, dtype)
        CLALibDropout.apply(x, 0.25, 11, 3, out=y)
        ref.close(y, want, bound)
        assert intact() and torch.equal(x, keep)
        CLALibDropout.apply(x, 0.25, 11, 3, out=x)
        assert torch.equal(x, y)
        x.fill_(float("nan"))
        assert bool(torch.isnan(flat).all())


def test_dropout_shards_draw_the_whole_mask_and_dropped_values_are_zero():
    x = normal(100, 333, torch.float32, 1)
    x[::3, ::2] = float("nan")
    x[1::3, ::5] = float("inf")
    whole = CLALibDropout.apply(x, 0.25, 11, 3)
    parts = torch.cat([CLALibDropout.apply(x[:37], 0.25, 11, 3), CLALibDropout.apply(x[37:], 0.25, 11, 3, row0=37)])
    assert torch.equal(whole.view(torch.int32), parts.view(torch.int32))
    f = ref.drop_factors(100, 333, 0.25, 11, 3)
    assert bool((whole.cpu()[f == 0] == 0).all())
    assert torch.equal(torch.isnan(whole).cpu(), torch.isnan(x).cpu() & (f != 0))
    y = x.clone()
    CLALibDropout.apply(y, 0.25, 11, 3, out=y)  # onto its own input
    assert torch.equal(y.view(torch.int32), whole.view(torch.int32))
    other = CLALibDropout.apply(torch.ones_like(x), 0.25, 11, 4)
    assert 0.2 < float((other == 0).float().mean()) < 0.3  # (33,300 draws: 0.05 is over 20 standard deviations)
    assert not torch.equal(other == 0, CLALibDropout.apply(torch.ones_like(x), 0.25, 11, 3) == 0)
    assert CLALibDropout.apply(x[:0], 0.5, 1).shape == (0, 333)


# ---- 8 bits ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows,cols,pad", [(1, 1, 0), (5, 7, 0), (1, 4096, 0), (200, 501, 0), (149, 2048, 8), (3, 20001, 0), (300, 33, 3)])
def test_quantize(dtype, rows, cols, pad):
    x = normal(rows, cols, dtype, rows * cols, pad=pad)
    x[rows // 2, :] = 0
    if rows > 4:
        x[0, cols // 2] = float("inf")
        x[1, cols - 1] = float("nan")
        x[2] *= 1e-6
    q, s = CLALibQ8.quantizeRows(x)
    wq, ws = ref.quantize(x)
    assert np.array_equal(q.cpu().numpy(), wq) and np.array_equal(s.cpu().numpy(), ws, equal_nan=True)
    q, s = CLALibQ8.quantizeCols(x)
    wq, ws = ref.quantize(x.t())
    assert np.array_equal(q.cpu().numpy(), wq) and np.array_equal(s.cpu().numpy(), ws, equal_nan=True)


def test_quantize_ties_and_extremes():
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -2.5], [127e30, 1e30, -127e30, 0, 0, 0], [1e-44, 0, 0, 0, -1e-44, 0], [-3.0, 3, 1, 0, 0, 0]],
                     device="cuda")
    q, s = CLALibQ8.quantizeRows(x)
    wq, ws = ref.quantize(x)
    assert wq[0].tolist() == [127, 0, 2, 2, 0, -2]
    assert np.array_equal(q.cpu().numpy(), wq) and np.array_equal(s.cpu().numpy(), ws)


def q8_want(a, sa, b, sb):
    return torch.from_numpy(a.astype(np.int64) @ b.astype(np.int64).T).double() * torch.from_numpy(sa).double()[:, None] * torch.from_numpy(sb).double()


def q8_bound(want, dtype):
    # FP64: two products; else the sum, the scales' product with it (three roundings of 2^-24), and the type's own
    return want.abs() * (2.0 ** -51 if dtype == torch.float64 else 2.0 ** -22 + ref.half_step(dtype)) + ref.tiny(dtype)


Q8_SIZES = [(1, 1, 1), (1, 64, 4096), (1, 129, 100), (7, 300, 501), (16, 128, 128), (33, 65, 31), (128, 128, 127), (129, 257, 129), (300, 1000, 640),
            (1000, 64, 16), (513, 2049, 1003), (2, 5000, 2048), (700, 511, 300)]


@pytest.mark.parametrize("M,N,K", Q8_SIZES)
@pytest.mark.parametrize("dtype", FLOATS)
def test_q8_product(M, N, K, dtype):
    rng = np.random.default_rng(M * N + K)
    a, b = rng.integers(-128, 128, (M, K), dtype=np.int8), rng.integers(-128, 128, (N, K), dtype=np.int8)
    sa, sb = rng.random(M, dtype=np.float32) + 0.1, (rng.random(N, dtype=np.float32) + 0.1) * 1e-3
    want = q8_want(a, sa, b, sb)
    dev = lambda v: torch.from_numpy(v).cuda()  # noqa: E731
    for lay in (0, 16, 5):  # contiguous; rows on 16-byte boundaries inside wider ones; anywhere
        wide = lambda v: torch.full((v.shape[0] + 1, -(-v.shape[1] // 16) * 16 + 2 * lay), 99, dtype=torch.int8, device="cuda")  # noqa: E731
        ta, tb = dev(a), dev(b)
        if lay:
            wa, wb = wide(a), wide(b)
            wa[:M, lay:lay + K], wb[:N, lay:lay + K] = ta, tb
            ta, tb = wa[:M, lay:lay + K], wb[:N, lay:lay + K]
        out, intact = framed(M, N, dtype)
        CLALibQ8.matrixMult(ta, dev(sa), tb, dev(sb), dtype, out=out)
        ref.close(out, want, q8_bound(want, dtype), f"layout {lay}")
        assert intact()
    again = CLALibQ8.matrixMult(ta, dev(sa), tb, dev(sb), dtype)
    assert torch.equal(again, out)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("pad", [0, 3])
@pytest.mark.parametrize("M,N,K", [(1, 64, 4096), (5, 77, 501), (200, 130, 333), (2, 3, 0), (1, 20000, 300), (16, 130, 256), (1, 300, 16), (3, 129, 1001),
                                   (1, 2000, 8192), (17, 40, 200)])
def test_q8_linear(M, N, K, dtype, pad):
    x, w = normal(M, K, dtype, 3, pad=pad), normal(K, N, torch.float32, 4)
    b, sb = CLALibQ8.quantizeCols(w)
    qa, sa = ref.quantize(x)
    want = q8_want(qa, sa, b.cpu().numpy(), sb.cpu().numpy())
    ref.close(CLALibQ8.linear(x, b, sb), want, q8_bound(want, dtype))
    if K:
        x[0, 0] = float("nan")
        y = CLALibQ8.linear(x, b, sb, dtype=torch.float32)
        assert bool(torch.isnan(y[0]).all()) and not bool(torch.isnan(y[1:]).any())


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("pad", [0, 3, 16])
@pytest.mark.parametrize("M,N,K", [(17, 1, 1), (300, 32, 100), (2500, 64, 501), (5000, 33, 128), (20011, 10, 20), (150, 256, 500), (1999, 200, 129),
                                   (700, 64, 1024), (40, 256, 1100), (2300, 64, 640), (333, 100, 700), (5000, 16, 1000)])
def test_q8_scores(M, N, K, dtype, pad):
    """Many rows against few columns, rows of zeros, of an infinity, of a NaN and of tiny values among them."""
    x, w = normal(M, K, dtype, 3, pad=pad), normal(K, N, torch.float32, 4)
    x[M // 3], x[M // 2, K // 2], x[M - 2, K - 1] = 0, float("inf"), float("nan")
    x[M - 1] *= 1e-6
    b, sb = CLALibQ8.quantizeCols(w)
    qa, sa = ref.quantize(x)
    out, intact = framed(M, N, dtype)
    CLALibQ8.linear(x, b, sb, out=out)
    bad = torch.tensor([M // 2, M - 2])
    good = torch.ones(M, dtype=torch.bool)
    good[bad] = False
    want = q8_want(qa[good], sa[good], b.cpu().numpy(), sb.cpu().numpy())
    ref.close(out[good.cuda()], want, q8_bound(want, dtype))
    assert intact() and bool(torch.isnan(out[bad.cuda()]).all())
    whole = CLALibQ8.linear(x, b, sb)
    assert torch.equal(whole[good.cuda()], out[good.cuda()])


def test_q8_largest_sums():
    """The longest sums that are taken, every term at its largest: -128 * -128 * 131071 = 2^31 - 2^14."""
    K = 131071
    a = torch.full((2, K), -128, dtype=torch.int8, device="cuda")
    a[1] = 127
    b = torch.full((130, K), -128, dtype=torch.int8, device="cuda")
    one = lambda n: torch.ones(n, device="cuda")  # noqa: E731
    out = CLALibQ8.matrixMult(a, one(2), b, one(130), torch.float64)
    assert bool((out[0] == 16384.0 * K).all()) and bool((out[1] == -127.0 * 128 * K).all())
    with pytest.raises(CLAError):
        wide = torch.zeros((1, K + 1), dtype=torch.int8, device="cuda")
        CLALibQ8.matrixMult(wide, one(1), wide, one(1))


# ---- the gated block ------------------------------------------------------------------------------------------------
GATED_SIZES = [(1, 1, 1), (1, 64, 128), (1, 100, 1000), (3, 33, 65), (17, 128, 130), (64, 256, 512), (128, 129, 257), (200, 72, 300), (513, 320, 200),
               (300, 1001, 731), (1000, 64, 40)]


def gated_inputs(M, D, F, dtype, pad=0, trans=False, packed=False):
    x = normal(M, D, dtype, M + D, pad=pad)
    if trans:
        wg, wu = normal(F, D, dtype, 5, D ** -0.5, pad).t(), normal(F, D, dtype, 6, D ** -0.5, pad).t()
    elif packed:
        w = normal(D, 2 * F, dtype, 5, D ** -0.5, pad)
        wg, wu = w[:, :F], w[:, F:]
    else:
        wg, wu = normal(D, F, dtype, 5, D ** -0.5, pad), normal(D, F, dtype, 6, D ** -0.5, pad)
    return x, wg, wu


@pytest.mark.parametrize("M,D,F", GATED_SIZES)
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("lay", ["plain", "padded", "packed", "trans"])
def test_gated_forward(M, D, F, dtype, lay):
    i = GATED_SIZES.index((M, D, F))
    act, p = ref.ACTS[i % 5], (0.0, 0.2)[i % 2]
    x, wg, wu = gated_inputs(M, D, F, dtype, 16 if lay == "padded" else 7 if lay == "packed" else 0, lay == "trans", lay == "packed")
    f = ref.drop_factors(M, F, p, 9, 4, 100)
    want, bound = ref.gated(x, wg, wu, act, f, dtype)
    h, intact = framed(M, F, dtype)
    got = CLALibGated.forward(x, wg, wu, act, p=p, seed=9, step=4, row0=100, save=True, out=h)
    for name, y, v, e in zip("hgu", got, want, bound):
        ref.close(y, v, e, name)
    assert intact()
    alone = CLALibGated.forward(x, wg, wu, act, p=p, seed=9, step=4, row0=100)
    assert torch.equal(alone, h)


@pytest.mark.parametrize("act", ref.ACTS)
@pytest.mark.parametrize("M", [1, 40, 300])
def test_gated_activations(act, M):
    x, wg, wu = gated_inputs(M, 64, 128, torch.bfloat16)
    wg = wg * 6  # gates far out on both sides
    f = torch.ones(M, 128, dtype=torch.float64)
    want, bound = ref.gated(x, wg, wu, act, f, torch.bfloat16)
    g, u, dh = want[1].to(torch.bfloat16).cuda(), want[2].to(torch.bfloat16).cuda(), normal(M, 128, torch.bfloat16, 8)
    ref.close(CLALibGated.forward(x, wg, wu, act), want[0], bound[0])
    want, bound = ref.gated_grads(dh, x, wg, wu, g, u, act, f, torch.bfloat16)
    for name, y, v, e in zip(("dx", "dwg", "dwu"), CLALibGated.backward(dh, x, wg, wu, g, u, act), want, bound):
        ref.close(y, v, e, name)


@pytest.mark.parametrize("M,D,F", GATED_SIZES)
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("lay", ["plain", "padded", "packed", "trans"])
def test_gated_backward(M, D, F, dtype, lay):
    i = GATED_SIZES.index((M, D, F))
    act, p = ref.ACTS[i % 5], (0.2, 0.0)[i % 2]
    pad = 16 if lay == "padded" else 7 if lay == "packed" else 0
    x, wg, wu = gated_inputs(M, D, F, dtype, pad, lay == "trans", lay == "packed")
    g, u, dh = (normal(M, F, dtype, s, pad=pad) for s in (11, 12, 13))
    f = ref.drop_factors(M, F, p, 9, 4)
    want, bound = ref.gated_grads(dh, x, wg, wu, g, u, act, f, dtype)
    got = CLALibGated.backward(dh, x, wg, wu, g, u, act, p=p, seed=9, step=4)
    for name, y, v, e in zip(("dx", "dwg", "dwu"), got, want, bound):
        ref.close(y, v, e, name)
    dx, none, _ = CLALibGated.backward(dh, x, wg, wu, g, u, act, p=p, seed=9, step=4, needW=False)
    assert none is None and torch.equal(dx, got[0])
    none, dwg, dwu = CLALibGated.backward(dh, x, wg, wu, g, u, act, p=p, seed=9, step=4, needX=False)
    assert none is None and torch.equal(dwg, got[1]) and torch.equal(dwu, got[2])


@pytest.mark.parametrize("act", ref.ACTS)
def test_gated_gradients_against_differences(act):
    """Central differences of the whole block in 64 bits, next to what forward saves and backward makes of it."""
    x, wg, wu = gated_inputs(6, 24, 32, torch.float16)
    dh = normal(6, 32, torch.float16, 3)
    h, g, u = CLALibGated.forward(x, wg, wu, act, p=0.25, seed=2, step=1, save=True)
    got = CLALibGated.backward(dh, x, wg, wu, g, u, act, p=0.25, seed=2, step=1)
    f = ref.drop_factors(6, 32, 0.25, 2, 1)
    v = [t.double().cpu() for t in (x, wg, wu)]
    loss = lambda: float((ref.act(act, v[0] @ v[1]) * (v[0] @ v[2]) * f * dh.double().cpu()).sum())  # noqa: E731
    rng = np.random.default_rng(0)
    for k, grad in enumerate(got):
        for _ in range(12):
            at = tuple(int(rng.integers(n)) for n in grad.shape)
            keep, step = float(v[k][at]), 1e-4
            v[k][at] = keep + step
            up = loss()
            v[k][at] = keep - step
            down = loss()
            v[k][at] = keep
            # fp16 products of 24 to 64 terms of order 1, each with half a step of 2^-11 in g, u, dg and the result; relu's kink lies within
            # `step` of a gate for none of these 192 gates but by chance, and then moves a term by step at most
            assert abs(float(grad[at]) - (up - down) / (2 * step)) < 0.02 * (1 + abs(float(grad[at])))


def test_gated_zero_sizes():
    for M, D, F in ((0, 16, 32), (4, 0, 32), (4, 16, 0)):
        x, w = torch.ones((M, D), dtype=torch.bfloat16, device="cuda"), torch.ones((D, F), dtype=torch.bfloat16, device="cuda")
        h, g, u = CLALibGated.forward(x, w, w, save=True)
        assert h.shape == (M, F) and not h.any() and not g.any()
        dx, dwg, dwu = CLALibGated.backward(h, x, w, w, g, u)
        assert dx.shape == (M, D) and dwg.shape == (D, F) and not dx.any() and not dwg.any() and not dwu.any()


def test_gated_values_that_are_not_finite_stay_in_their_rows():
    x, wg, wu = gated_inputs(70, 64, 96, torch.bfloat16)
    clean = CLALibGated.forward(x, wg, wu)
    x[3, 5] = float("nan")
    x[40, 0] = float("inf")
    h = CLALibGated.forward(x, wg, wu, p=0.5, seed=3)
    f = ref.drop_factors(70, 96, 0.5, 3)
    assert bool((h.cpu()[f == 0] == 0).all()) and bool(torch.isnan(h[3].cpu()[f[3] != 0]).all())
    rest = [r for r in range(70) if r not in (3, 40)]
    assert torch.equal(CLALibGated.forward(x, wg, wu)[rest], clean[rest])


@pytest.mark.parametrize("act", ref.ACTS)
def test_gated_slopes_of_large_gates(act):
    """Where the square or the cube of a gate leaves FP32 the slope is that of the line: 1 or 0."""
    g = torch.tensor([[1e38, -1e38, 1e20, -1e20, 1e13, -1e13, 200.0, -200.0]], dtype=torch.bfloat16, device="cuda")
    one = torch.ones_like(g)
    w = torch.ones((8, 8), dtype=torch.bfloat16, device="cuda")
    _, dwg, dwu = CLALibGated.backward(one, one, w, w, g, one, act, needX=False)
    up = (g > 0).to(g.dtype)
    assert torch.equal(dwg, (torch.zeros_like(up) if act == "sigmoid" else up).expand(8, 8))
    assert torch.equal(dwu, (up if act == "sigmoid" else up * g).expand(8, 8))


MANY = [(2500, 1100, 3001), (40, 5000, 9000), (300, 6000, 260), (1, 3000, 20000), (700, 2050, 1800), (32, 8200, 520)]


@pytest.mark.parametrize("M,D,F", MANY)
@pytest.mark.parametrize("dtype", HALVES)
def test_gated_of_many_tiles(M, D, F, dtype):
    """More tiles than SMs, depths that several CTAs share, and sums over many stages (the 64-bit forms on the GPU)."""
    x, wg, wu = gated_inputs(M, D, F, dtype)
    f = ref.drop_factors(M, F, 0.1, 21, 5).cuda()
    want, bound = ref.gated(x, wg, wu, "silu", f, dtype, "cuda")
    got = CLALibGated.forward(x, wg, wu, "silu", p=0.1, seed=21, step=5, save=True)
    for name, y, v, e in zip("hgu", got, want, bound):
        ref.close(y, v, e, name)
    dh = normal(M, F, dtype, 13)
    want, bound = ref.gated_grads(dh, x, wg, wu, got[1], got[2], "silu", f, dtype, "cuda")
    grads = CLALibGated.backward(dh, x, wg, wu, got[1], got[2], "silu", p=0.1, seed=21, step=5)
    for name, y, v, e in zip(("dx", "dwg", "dwu"), grads, want, bound):
        ref.close(y, v, e, name)
    for _ in range(3):  # bit by bit the same, whatever ran before
        again = CLALibGated.backward(dh, x, wg, wu, got[1], got[2], "silu", p=0.1, seed=21, step=5)
        assert all(torch.equal(p, q) for p, q in zip(again, grads))


@pytest.mark.parametrize("M,N,K", [(3000, 5001, 700), (16, 9000, 4096), (100, 1000, 20000), (1, 20001, 1024), (5000, 64, 501), (260, 30000, 130)])
def test_q8_of_many_tiles(M, N, K):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(M + N)
    a, b = (torch.randint(-128, 128, s, dtype=torch.int8, device="cuda", generator=gen) for s in ((M, K), (N, K)))
    sa, sb = torch.rand(M, device="cuda", generator=gen) + 0.1, torch.rand(N, device="cuda", generator=gen) + 0.1
    want = (a.double() @ b.double().T) * sa.double()[:, None] * sb.double()  # (whole sums below 2^53: exact)
    for dtype in FLOATS:
        got = CLALibQ8.matrixMult(a, sa, b, sb, dtype)
        # A rounding to the type gives an infinity from half a step above its largest value on (fp16: 65504 + 16 = 65520): there the definition
        # has one, and just there, within the FP32 scaling's 2^-22, either
        top = float(torch.finfo(dtype).max) * (1 + ref.half_step(dtype) / 2)
        over, under = want.abs() > top * (1 + 2.0 ** -22), want.abs() < top * (1 - 2.0 ** -22)
        assert torch.equal(got[over].double(), torch.copysign(torch.full_like(want[over], float("inf")), want[over]))
        ref.close(torch.where(under, got.double(), 0), torch.where(under, want, 0), q8_bound(want, dtype))
        assert torch.equal(got, CLALibQ8.matrixMult(a, sa, b, sb, dtype))


def test_offsets_beyond_32_bits():
    """Matrices of more than 2^31 elements: their last rows."""
    M, F = 70_001, 32_000
    x, wg, wu = gated_inputs(M, 64, F, torch.bfloat16)
    h = CLALibGated.forward(x, wg, wu, p=0.5, seed=3)
    f = ref.drop_factors(5, F, 0.5, 3, 0, M - 5)
    want, bound = ref.gated(x[-5:], wg, wu, "silu", f, torch.bfloat16)
    ref.close(h[-5:], want[0], bound[0])
    y = CLALibDropout.apply(h, 0.25, 9)
    f = ref.drop_factors(3, F, 0.25, 9, 0, M - 3)
    want = h[-3:].double().cpu() * f
    ref.close(y[-3:], want, want.abs() * (ref.half_step(torch.bfloat16) + 2.0 ** -22) + ref.tiny(torch.bfloat16))
    dx, _, _ = CLALibGated.backward(y, x, wg, wu, h, h, needW=False)
    want, bound = ref.gated_grads(y[-4:], x[-4:], wg, wu, h[-4:], h[-4:], "silu", torch.ones(4, F, dtype=torch.float64), torch.bfloat16)
    ref.close(dx[-4:], want[0], bound[0])
    del y, dx
    q, s = CLALibQ8.quantizeRows(h)
    wq, ws = ref.quantize(h[-3:])
    assert np.array_equal(q[-3:].cpu().numpy(), wq) and np.array_equal(s[-3:].cpu().numpy(), ws)
    del h
    b = torch.randint(-128, 128, (40, F), dtype=torch.int8, device="cuda")
    got = CLALibQ8.matrixMult(q, s, b, torch.ones(40, device="cuda"), torch.float64)
    want = q8_want(wq, ws, b.cpu().numpy(), np.ones(40, np.float32))
    ref.close(got[-3:], want, q8_bound(want, torch.float64))
    del q
    torch.cuda.empty_cache()


def test_scores_of_more_than_32_bits_of_values():
    M, K, N = 4_400_003, 500, 33
    x = torch.zeros((M, K), dtype=torch.bfloat16, device="cuda")
    at = [0, 1, M // 2, M - 700, M - 1]
    x[at] = normal(5, K, torch.bfloat16, 1)
    b, sb = CLALibQ8.quantizeCols(normal(K, N, torch.float32, 2))
    got = CLALibQ8.linear(x, b, sb)
    qa, sa = ref.quantize(x[at])
    want = q8_want(qa, sa, b.cpu().numpy(), sb.cpu().numpy())
    ref.close(got[at], want, q8_bound(want, torch.bfloat16))
    got[at] = 0
    assert not bool(got.any())
    del x, got
    torch.cuda.empty_cache()


def test_a_row_of_two_gigabytes_off_its_boundary():
    D = 1 << 30
    x = torch.zeros(D + 1, dtype=torch.bfloat16, device="cuda")[1:].reshape(1, D)
    w = [torch.zeros((2, D), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    for k, at in enumerate((0, 7, 12345, D // 2, D - 9, D - 1)):
        x[0, at] = 1
        w[0][:, at] = 1 << k
        w[1][1, at] = 1
    h = CLALibGated.forward(x, w[0].t(), w[1].t(), "relu")
    assert h.tolist() == [[0.0, 63 * 6.0]]
    del x, w, h
    torch.cuda.empty_cache()


# ---- beside one another -----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("M,D,F", [(64, 256, 512), (333, 1001, 2731), (3, 2000, 999)])
def test_streams_and_graphs(M, D, F):
    """Calls on two streams at once, and captured calls replayed in turn with direct ones."""
    x, wg, wu = gated_inputs(M, D, F, torch.bfloat16)
    w8, s8 = CLALibQ8.quantizeCols(normal(501, 64, torch.float32, 2))
    z = normal(M, 501, torch.float32, 1)
    dh = normal(M, F, torch.bfloat16, 4)

    def step():
        h, g, u = CLALibGated.forward(x, wg, wu, "gelu", p=0.1, seed=1, step=2, save=True)
        return (h,) + CLALibGated.backward(dh, x, wg, wu, g, u, "gelu", p=0.1, seed=1, step=2)

    def score():
        return (CLALibQ8.linear(z, w8, s8), CLALibDropout.apply(z, 0.5, 3))

    want, scores = step(), score()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        with torch.cuda.stream(a):
            got = [step() for _ in range(6)]
        with torch.cuda.stream(b):
            sc = [score() for _ in range(12)]
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for r in got for p, q in zip(r, want))
        assert all(torch.equal(p, q) for r in sc for p, q in zip(r, scores))
    graphs = []
    for f in (step, score, step):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = f()
        graphs.append((graph, out))
    for t in (t for _, out in graphs for t in out):
        t.zero_()
    for graph, _ in graphs * 2:
        graph.replay()
    direct = step()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for (_, out), w in zip(graphs, (want, scores, want)) for p, q in zip(out, w))
    assert all(torch.equal(p, q) for p, q in zip(direct, want))


def test_compressed_block_through_the_layers():
    """A compressed block's rows through a hidden layer with dropout, its gradients, and its scores in 8 bits."""
    cmb = datagen.random_cmb(3, 5000, datagen.KINDS).to_device(0)
    X = torch.from_numpy(dense_of(cmb))
    n, m = X.shape
    for r0, rows in ((0, 5000), (1000, 1500), (4999, 1), (1024, 1024), (77, 0)):
        for dtype in FLOATS:
            part = CLALibDecompress.rows(cmb, r0, rows, dtype)
            want = X[r0:r0 + rows]
            ref.close(part, want, want.abs() * (2.0 ** -50 + ref.half_step(dtype)) + ref.tiny(dtype) + 1e-14)
    wide = torch.full((300, m + 9), 7.0, device="cuda", dtype=torch.bfloat16)
    CLALibDecompress.rows(cmb, 100, 300, torch.bfloat16, out=wide[:, 4:4 + m])
    assert bool((wide[:, :4] == 7).all()) and bool((wide[:, 4 + m:] == 7).all())
    x = wide[:, 4:4 + m]
    wg, wu = normal(m, 40, torch.bfloat16, 1, m ** -0.5), normal(m, 40, torch.bfloat16, 2, m ** -0.5)
    h, g, u = CLALibGated.forward(x, wg, wu, "gelu", p=0.1, seed=5, row0=100, save=True)
    f = ref.drop_factors(300, 40, 0.1, 5, 0, 100)
    want, bound = ref.gated(x, wg, wu, "gelu", f, torch.bfloat16)
    ref.close(h, want[0], bound[0])
    dh = normal(300, 40, torch.bfloat16, 6)
    want, bound = ref.gated_grads(dh, x, wg, wu, g, u, "gelu", f, torch.bfloat16)
    for y, v, e in zip(CLALibGated.backward(dh, x, wg, wu, g, u, "gelu", p=0.1, seed=5, row0=100), want, bound):
        ref.close(y, v, e)
    b, sb = CLALibQ8.quantizeCols(normal(m, 33, torch.float64, 9))
    got = CLALibQ8.rightMultByMatrix(cmb, b, sb)
    assert torch.equal(got, CLALibQ8.linear(CLALibDecompress.rows(cmb, 0, 5000, torch.float64), b, sb))
    qa, sa = ref.quantize(X)
    want = q8_want(qa, sa, b.cpu().numpy(), sb.cpu().numpy())
    # (a cell whose sum of groups rounds otherwise may take the next whole number: one step of its row's scale times one of the weights)
    ref.close(got, want, 1e-9 + 130 * torch.from_numpy(sa).double()[:, None] * sb.cpu().double())
    with pytest.raises(CLAError):
        CLALibDecompress.rows(cmb, 4000, 1001, torch.float32)
    with pytest.raises(CLAError):
        CLALibQ8.rightMultByMatrix(cmb, b[:, 1:], sb)
    cmb.free()


@pytest.mark.parametrize("N", [5, 140, 300])
def test_scores_of_a_block_in_the_smallest_chunks(N):
    """Chunks of 1024 rows, the last of nine: the same results as in one, in every type."""
    cmb = datagen.random_cmb(4, 2 * 1024 + 9, datagen.KINDS).to_device(0)
    n, m = 2 * 1024 + 9, cmb.clen
    b, sb = CLALibQ8.quantizeCols(normal(m, N, torch.float64, 9))
    rows = CLALibDecompress.rows(cmb, 0, n, torch.float64)
    up = lambda v: -(-v // 256) * 256  # noqa: E731
    pitch = -(-m // 128) * 128
    size = up(1024 * pitch) + up(1024 * 4) + up(1024 * m * 8) + up(N * pitch)
    L = native.lib()
    for code, dtype in enumerate(FLOATS):
        out, intact = framed(n, N, dtype)
        work = torch.empty(size, dtype=torch.uint8, device="cuda")
        call = lambda bytes: L.cla_q8_rmm_dev(cmb.handle(), b.data_ptr(), b.stride(0), sb.data_ptr(), N, code, out.data_ptr(), out.stride(0),  # noqa: E731
                                              work.data_ptr(), bytes, torch.cuda.current_stream().cuda_stream)
        with pytest.raises(CLAError):
            native.check(call(size // 2))
        native.check(call(size))
        assert torch.equal(out, CLALibQ8.linear(rows, b, sb, dtype=dtype)) and intact()
    cmb.free()


def test_refusals_on_the_device():
    x, wg, wu = gated_inputs(8, 16, 32, torch.bfloat16)
    q, s = CLALibQ8.quantizeRows(x)
    for f in (lambda: CLALibGated.forward(x, wg, wu.half()), lambda: CLALibGated.forward(x, wg, wu[:, :31]), lambda: CLALibGated.forward(x.float(), wg, wu),
              lambda: CLALibGated.forward(x, wg, wu, "tanh"), lambda: CLALibGated.forward(x.t().contiguous().t(), wg, wu),
              lambda: CLALibGated.forward(x, wg, wu, p=1.0), lambda: CLALibGated.forward(x, wg, wu, seed=-1),
              lambda: CLALibGated.forward(x, wg, wu, out=x), lambda: CLALibGated.backward(wg, x, wg, wu, wg, wu),
              lambda: CLALibQ8.matrixMult(q, s, q[:, :15], s), lambda: CLALibQ8.matrixMult(q, s[:7], q, s), lambda: CLALibQ8.matrixMult(q, None, q, s),
              lambda: CLALibQ8.matrixMult(q, s, q, s, torch.int32), lambda: CLALibQ8.matrixMult(q, s, q, s, out=torch.empty(8, 7, device="cuda")),
              lambda: CLALibQ8.quantizeRows(q), lambda: CLALibDropout.apply(x[0], 0.5, 1), lambda: CLALibDropout.apply(x, 1.5, 1),
              lambda: CLALibDropout.apply(x, 0.5, 1, out=torch.empty_like(x).half()), lambda: CLALibDropout.apply(x[:1].expand(8, 16), 0.5, 1, out=x)):
        with pytest.raises(CLAError):
            f()


def test_a_refused_device_leaves_the_next_call_as_it_was():
    x = normal(8, 16, torch.float32, 1)
    y, d = torch.empty_like(x), native.cla_drop(0.5, 1, 2, 0)
    with pytest.raises(CLAError):
        native.check(native.lib().cla_dropout_dev(1, x.data_ptr(), 16, 8, 16, y.data_ptr(), 16, C.byref(d), 99, None))
    assert torch.equal(CLALibDropout.apply(x, 0.5, 1, 2, out=y), CLALibDropout.apply(x, 0.5, 1, 2))
    for f in (lambda: CLALibDropout.apply(x, 0.5, 1, row0=(1 << 64) + 5), lambda: CLALibDropout.apply(x, 0.5, 1, out=[1]),
              lambda: CLALibDropout.apply(x, 0.5, 1, out=y.cpu().numpy())):
        with pytest.raises(CLAError):
            f()


def test_status_waits_for_every_stream():
    x = torch.ones((8192, 8192), device="cuda")
    y = torch.empty_like(x)
    CLALibDropout.apply(x, 0.5, 1, out=y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for step in range(100):
            CLALibDropout.apply(x, 0.5, 1, step, out=y)
    status()
    assert side.query()
