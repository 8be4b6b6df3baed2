"""Dense operators beside the compressed products, on device tensors: what a model does with a product's result.

* ``CLALibQ8``       products in 8-bit integers with a scale per row of the left operand and per column of the right one, and the quantiser
* ``CLALibGated``    the gated feed-forward block ``act(X Wg) * (X Wu)`` and its gradients
* ``CLALibDropout``  dropout from a counter-based generator; nothing of the mask is stored

They have no counterpart in the reference. Operands are torch CUDA tensors with rows of adjacent elements (any row stride; weights may also be
transposed views). Each call is enqueued on the current stream of its tensors' device, takes results and workspaces from torch's
allocator, and may be captured into a graph. Nothing is recorded for autograd: gradients are the ``backward`` calls' and the dropout's own. An ``out`` that
shares memory with an operand is refused, but for dropout onto its own input. A ``CompressedMatrixBlock`` takes part through
``CLALibQ8.rightMultByMatrix`` and ``CLALibDecompress.rows``. Failures raise ``CLAError``.
"""
from __future__ import annotations

import ctypes as C
from operator import index

import torch

from . import native
from .cmb import CompressedMatrixBlock
from .native import CLAError, check

TYPES = {torch.float64: 0, torch.float32: 1, torch.bfloat16: 2, torch.float16: 3}
ACTS = {"silu": 0, "gelu": 1, "gelu_tanh": 2, "relu": 3, "sigmoid": 4}


def _stream(index: int) -> int:
    return torch._C._cuda_getCurrentRawStream(index)


def _fail(code: int, msg: str):
    raise CLAError(code, msg)


def _rows(t, what: str, dtype=None, device: int = -1):
    """Address and row stride of a device matrix whose rows have adjacent elements."""
    try:
        dev = t.get_device()
        rows, cols = t.shape
        s0, s1 = t.stride()
    except (AttributeError, ValueError, RuntimeError):
        if not isinstance(t, torch.Tensor):
            _fail(-2, f"{what}: a CUDA tensor is needed")
        _fail(-4, f"{what}: two dimensions are needed")
    if dev < 0:
        _fail(-2, f"{what}: a CUDA tensor is needed")
    if dtype is not None and t.dtype != dtype:
        _fail(-3, f"{what}: type {t.dtype}, expected {dtype}")
    if device >= 0 and dev != device:
        _fail(-2, f"{what}: on another device than the first operand")
    if s1 != 1 and cols > 1:
        _fail(-3, f"{what}: the elements of a row must be adjacent")
    if rows <= 1:
        s0 = cols
    elif s0 < cols:
        _fail(-4, f"{what}: rows overlap")
    return t.data_ptr(), s0


def _vector(t, what: str, n: int, device: int):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.get_device() != device:
        _fail(-2, f"{what}: float32 on the operands' device is needed")
    if t.dim() != 1 or t.shape[0] != n or (n > 1 and t.stride(0) != 1):
        _fail(-4, f"{what}: {n} adjacent values are needed")
    return t.data_ptr()


def _result(out, shape, dtype, like, what: str):
    """``out``, or a new tensor on the device of ``like``."""
    if out is None:
        return like.new_empty(shape) if like.dtype == dtype else torch.empty(shape, dtype=dtype, device=like.device)
    if not isinstance(out, torch.Tensor):
        _fail(-2, f"{what}: a CUDA tensor is needed")
    if out.shape != shape:
        _fail(-4, f"{what}: shape {tuple(out.shape)}, expected {tuple(shape)}")
    return out


def _type(dtype, what: str) -> int:
    t = TYPES.get(dtype) if isinstance(dtype, torch.dtype) else None
    if t is None:
        _fail(-3, f"{what}: unsupported type {dtype}")
    return t


def _workspace(n: int, device):
    return torch.empty(n, dtype=torch.uint8, device=device)


def _workspace_like(n: int, t):
    """The same, by the quicker way where a tensor is at hand."""
    return t.new_empty(-(-n // t.element_size()))


def _drop(p, seed, step, row0) -> native.cla_drop:
    try:
        return _drop_of(p, seed, step, row0)
    except (TypeError, OverflowError):  # (numbers of other kinds than Python's own)
        pass
    try:
        p, seed, step, row0 = float(p * 1.0), index(seed), index(step), index(row0)
    except (TypeError, ValueError):
        _fail(-2, "dropout: p is a number, seed, step and row0 are whole numbers")
    return _drop_of(p, seed, step, row0)


def _drop_of(p, seed, step, row0) -> native.cla_drop:
    if not 0 <= seed < 1 << 64 or not 0 <= step < 1 << 64:
        _fail(-2, "dropout: seed and step are unsigned 64-bit numbers")
    if not 0 <= row0 <= 1 << 32:
        _fail(-2, "dropout: rows beyond 2^32")
    return native.cla_drop(p, seed, step, row0)


class CLALibDropout:
    @staticmethod
    def apply(x, p: float, seed: int, step: int = 0, row0: int = 0, out=None):
        """``x`` with each element zero with probability ``p``, else times ``1 / (1 - p)``. Word ``c % 4`` of Philox4x32-10 with key
        ``seed`` and counter ``(c / 4, row0 + r, step)`` decides about element (r, c): applied to the output's gradient with the same
        ``(seed, step)`` it is the backward pass, and a shard of rows passes its first row as ``row0``. ``out`` may be ``x`` itself."""
        px, ldx = _rows(x, "dropout, x")
        dtype = x.dtype
        t = _type(dtype, "dropout")
        dev = x.get_device()
        rows, cols = shape = x.shape
        y = _result(out, shape, dtype, x, "dropout, out")
        py, ldy = (y.data_ptr(), cols) if out is None else _rows(y, "dropout, out", dtype, dev)
        d = _drop(p, seed, step, row0)
        check(native.lib().cla_dropout_dev(t, px, ldx, rows, cols, py, ldy, C.byref(d), dev, _stream(dev)))
        return y


class CLALibQ8:
    @staticmethod
    def quantizeRows(x):
        """``(q, scale)``: int8 rows and a float32 scale per row, ``x ~ q * scale[:, None]`` (scale = largest magnitude / 127)."""
        px, ldx = _rows(x, "quantize, x")
        t = _type(x.dtype, "quantize")
        rows, cols = x.shape
        q = torch.empty((rows, -(-cols // 128) * 128), dtype=torch.int8, device=x.device)[:, :cols]
        scale = torch.empty(rows, dtype=torch.float32, device=x.device)
        dev = x.get_device()
        check(native.lib().cla_q8_quantize_dev(t, px, ldx, rows, cols, 0, q.data_ptr(), -(-cols // 128) * 128, scale.data_ptr(), dev, _stream(dev)))
        return q, scale

    @staticmethod
    def quantizeCols(w):
        """``(q, scale)`` of a weight matrix ``w`` [K x N], laid out for the products: q is [N x K], a row and a scale per column."""
        pw, ldw = _rows(w, "quantize, w")
        t = _type(w.dtype, "quantize")
        rows, cols = w.shape
        q = torch.empty((cols, -(-rows // 128) * 128), dtype=torch.int8, device=w.device)[:, :rows]
        scale = torch.empty(cols, dtype=torch.float32, device=w.device)
        dev = w.get_device()
        check(native.lib().cla_q8_quantize_dev(t, pw, ldw, rows, cols, 1, q.data_ptr(), -(-rows // 128) * 128, scale.data_ptr(), dev, _stream(dev)))
        return q, scale

    @staticmethod
    def _mm(a, aType, aScale, b, bScale, dtype, out):
        pa, lda = _rows(a, "8-bit product, a")
        dev = a.get_device()
        pb, ldb = _rows(b, "8-bit product, b", torch.int8, dev)
        M, K = a.shape
        N, inner = b.shape
        if inner != K:
            _fail(-4, "8-bit product: inner dimensions do not match")
        outType = _type(dtype, "8-bit product")
        y = _result(out, (M, N), dtype, a, "8-bit product, out")
        py, ldo = (y.data_ptr(), N) if out is None else _rows(y, "8-bit product, out", dtype, dev)
        L = native.lib()
        args = native.cla_q8(M, N, K, pa, lda, None if aScale is None else _vector(aScale, "8-bit product, scales of a", M, dev), pb, ldb,
                             _vector(bScale, "8-bit product, scales of b", N, dev), py, ldo, None, 0, aType, outType, dev)
        ref = C.byref(args)
        n = check(L.cla_q8_workspace(ref))
        if n:
            work = _workspace_like(n, a)
            args.work, args.workBytes = work.data_ptr(), n
        check(L.cla_q8_mm_dev(ref, _stream(dev)))
        return y

    @staticmethod
    def matrixMult(a, aScale, b, bScale, dtype=torch.float32, out=None):
        """``out[m, n] = aScale[m] * bScale[n] * sum_k a[m, k] * b[n, k]`` for int8 ``a`` [M x K] and ``b`` [N x K] (a row per output
        column, as ``quantizeCols`` gives), exact up to the scaling and one rounding to ``dtype``. ``out`` shares no memory with an operand."""
        if not isinstance(a, torch.Tensor) or a.dtype != torch.int8:
            _fail(-3, "8-bit product: a must be int8")
        if aScale is None:
            _fail(-2, "8-bit product: scales of a are needed")
        return CLALibQ8._mm(a, 4, aScale, b, bScale, dtype, out)

    @staticmethod
    def linear(x, b, bScale, dtype=None, out=None):
        """``x %*% W`` with W in 8 bits (``b``, ``bScale`` of ``quantizeCols(W)``): the rows of ``x`` are quantised in the call.
        The result has the type of ``x`` unless ``dtype`` says otherwise; ``out`` shares no memory with an operand."""
        if not isinstance(x, torch.Tensor):
            _fail(-2, "8-bit product, x: a CUDA tensor is needed")
        return CLALibQ8._mm(x, _type(x.dtype, "8-bit product"), None, b, bScale, x.dtype if dtype is None else dtype, out)

    @staticmethod
    def rightMultByMatrix(m1, b, bScale, dtype=torch.float64, out=None):
        """``m1 %*% W`` for a compressed block ``m1`` and W in 8 bits, as ``linear`` of its rows (beside
        ``CLALibRightMultBy.rightMultByMatrix``, in FP64). The result is a tensor on the block's device."""
        if not isinstance(m1, CompressedMatrixBlock):
            _fail(-2, "8-bit right product, m1: a compressed block is needed")
        dev = m1.device if m1.device is not None else 0
        pb, ldb = _rows(b, "8-bit right product, b", torch.int8, dev)
        N = b.shape[0]
        if b.shape[1] != m1.clen:
            _fail(-4, "8-bit right product: inner dimensions do not match")
        ps = _vector(bScale, "8-bit right product, scales", N, dev)
        outType = _type(dtype, "8-bit right product")
        y = _result(out, (m1.rlen, N), dtype, b, "8-bit right product, out")
        py, ldo = _rows(y, "8-bit right product, out", dtype, dev)
        L = native.lib()
        n = check(L.cla_q8_rmm_workspace(m1.handle(), N))
        work = _workspace(n, b.device)
        check(L.cla_q8_rmm_dev(m1.handle(), pb, ldb, ps, N, outType, py, ldo, work.data_ptr(), n, _stream(dev)))
        return y


class CLALibGated:
    """``H = dropout(act(X Wg) * (X Wu))`` in bfloat16 or float16 with sums in FP32, and its gradients. ``act``: "silu", "gelu" (erf),
    "gelu_tanh", "relu" or "sigmoid". Weights [D x F], or transposed views of [F x D] tensors (both alike). Nothing is recorded for autograd, also
    where operands require gradients: they are what ``backward`` returns."""

    @staticmethod
    def _args(x, wGate, wUp, act, p, seed, step, row0):
        px, ldx = _rows(x, "gated block, x")
        dev = x.get_device()
        if x.dtype != torch.bfloat16 and x.dtype != torch.float16:
            _fail(-3, f"gated block: unsupported type {x.dtype} (bfloat16 and float16)")
        a = ACTS.get(act) if isinstance(act, str) else None
        if a is None:
            _fail(-3, f"gated block: unknown activation {act!r}")
        M, D = x.shape
        trans = 0
        for w, what in ((wGate, "gated block, wGate"), (wUp, "gated block, wUp")):
            if not isinstance(w, torch.Tensor) or w.dim() != 2:
                _fail(-2, what + ": a CUDA matrix is needed")
        if wGate.shape[0] != D or wGate.shape != wUp.shape:
            _fail(-4, "gated block: weights must both be [columns of x, F]")
        if wGate.stride(1) != 1 and wGate.shape[1] > 1:
            wGate, wUp, trans = wGate.t(), wUp.t(), 1
        pg, ldg = _rows(wGate, "gated block, wGate", x.dtype, dev)
        pu, ldu = _rows(wUp, "gated block, wUp", x.dtype, dev)
        c = native.cla_gated(M, D, wGate.shape[0] if trans else wGate.shape[1], px, pg, pu, ldx, ldg, ldu)
        c.drop = _drop(p, seed, step, row0)
        c.type, c.act, c.wTrans, c.device = TYPES[x.dtype], a, trans, dev
        return c

    @staticmethod
    def _run(c, backward, x):
        L, ref = native.lib(), C.byref(c)
        n = check(L.cla_gated_workspace(ref, backward))
        if n:
            work = _workspace_like(n, x)
            c.work, c.workBytes = work.data_ptr(), n
        check((L.cla_gated_bwd_dev if backward else L.cla_gated_fwd_dev)(ref, _stream(c.device)))

    @staticmethod
    def forward(x, wGate, wUp, act: str = "silu", p: float = 0.0, seed: int = 0, step: int = 0, row0: int = 0, save: bool = False, out=None):
        """``H`` [rows of x, F]; with ``save`` also ``X Wg`` and ``X Wu``, which ``backward`` takes. ``p``, ``seed``, ``step``, ``row0``:
        dropout of H, as ``CLALibDropout.apply``. ``out`` shares no memory with an operand."""
        c = CLALibGated._args(x, wGate, wUp, act, p, seed, step, row0)
        h = _result(out, (c.M, c.F), x.dtype, x, "gated block, out")
        c.h, c.ldh = (h.data_ptr(), c.F) if out is None else _rows(h, "gated block, out", x.dtype, c.device)
        if save:
            g, u = x.new_empty((c.M, c.F)), x.new_empty((c.M, c.F))
            c.g, c.u = g.data_ptr(), u.data_ptr()
            c.ldg = c.ldu = c.F
        CLALibGated._run(c, 0, x)
        return (h, g, u) if save else h

    @staticmethod
    def backward(dH, x, wGate, wUp, g, u, act: str = "silu", p: float = 0.0, seed: int = 0, step: int = 0, row0: int = 0, needX: bool = True,
                 needW: bool = True):
        """``(dX, dWg, dWu)`` from the gradient of H and what ``forward(..., save=True)`` gave, with the same activation and dropout
        arguments; dX or the weights' gradients are None where not needed."""
        c = CLALibGated._args(x, wGate, wUp, act, p, seed, step, row0)
        dev, M, F = c.device, c.M, c.F
        for t, what in ((dH, "dH"), (g, "g"), (u, "u")):
            if not isinstance(t, torch.Tensor) or t.shape != (M, F):
                _fail(-4, f"gated block, {what}: expected [{M}, {F}]")
        c.dh, c.lddh = _rows(dH, "gated block, dH", x.dtype, dev)
        c.g, c.ldg = _rows(g, "gated block, g", x.dtype, dev)
        c.u, c.ldu = _rows(u, "gated block, u", x.dtype, dev)
        dx = dwg = dwu = None
        if needX:
            dx = x.new_empty((c.M, c.D))
            c.dx, c.lddx = dx.data_ptr(), c.D
        if needW:
            dwg, dwu = x.new_empty((c.D, c.F)), x.new_empty((c.D, c.F))
            c.dwg, c.dwu = dwg.data_ptr(), dwu.data_ptr()
            c.lddwg = c.lddwu = c.F
        CLALibGated._run(c, 1, x)
        return dx, dwg, dwu


def status(device: int = 0) -> None:
    """Waits for the device and raises ``CLAError`` (DEVICE_CHECK) if a kernel's self-check tripped in an earlier dense call."""
    check(native.lib().cla_dense_status(device))
