"""The dense operators without a GPU: the generator against published vectors, what the C entry points and the classes refuse."""
import ctypes as C

import numpy as np
import pytest
import torch

from systemds_b200 import CLAError, CLALibDropout, CLALibGated, CLALibQ8, native
from systemds_b200.native import check
from tests import dense_ref as ref

P = 1 << 20  # an address that nothing reads: the calls below are refused on the host


def test_philox_known_answers():
    """The vectors published with the generator."""
    f = 0xFFFFFFFF
    assert [int(v) for v in ref.philox(np.zeros(4, np.uint64), (0, 0))] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert [int(v) for v in ref.philox(np.full(4, f, np.uint64), (f, f))] == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    pi = np.array([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], np.uint64)
    assert [int(v) for v in ref.philox(pi, (0xA4093822, 0x299F31D0))] == [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


def refused(code, f):
    with pytest.raises(CLAError) as e:
        check(f())
    assert e.value.code == code, str(e.value)


def test_dropout_refusals():
    L = native.lib()

    def call(type=1, x=P, ldx=8, rows=4, cols=8, y=P, ldy=8, p=0.5, row0=0):
        return L.cla_dropout_dev(type, x, ldx, rows, cols, y, ldy, C.byref(native.cla_drop(p, 1, 2, row0)), 0, None)

    for code, kw in ((-3, {"type": 4}), (-3, {"type": 9}), (-4, {"rows": -1}), (-4, {"ldx": 7}), (-4, {"ldy": 7}), (-2, {"x": None}), (-2, {"y": None}),
                     (-2, {"p": 1.0}), (-2, {"p": -0.1}), (-2, {"p": float("nan")}), (-2, {"row0": -1}), (-2, {"row0": (1 << 32) - 3}),
                     (-2, {"x": P + 2}), (-3, {"rows": 1 << 31})):
        refused(code, lambda: call(**kw))
    refused(-2, lambda: L.cla_dropout_dev(1, P, 8, 4, 8, P, 8, None, 0, None))


def test_q8_refusals():
    L = native.lib()

    def args(**kw):
        c = native.cla_q8(M=4, N=4, K=16, a=P, lda=16, aScale=P, b=P, ldb=16, bScale=P, out=P, ldo=4, aType=4, outType=1, device=0)
        for k, v in kw.items():
            setattr(c, k, v)
        return C.byref(c)

    for code, kw in ((-3, {"aType": 7}), (-3, {"outType": 4}), (-3, {"K": 131072, "lda": 131072, "ldb": 131072}), (-4, {"M": -1}), (-4, {"lda": 15}),
                     (-4, {"ldb": 15}), (-4, {"ldo": 3}), (-2, {"a": None}), (-2, {"b": None}), (-2, {"out": None}), (-2, {"aScale": None}),
                     (-2, {"bScale": None}), (-2, {"out": P + 2}), (-2, {"aType": 0, "a": P + 4})):
        refused(code, lambda: L.cla_q8_mm_dev(args(**kw), None))
        refused(code, lambda: L.cla_q8_workspace(args(**kw)))
    assert L.cla_q8_workspace(args()) == 0
    assert L.cla_q8_workspace(args(K=15)) == 0  # (rows 16 bytes apart all the same)
    need = L.cla_q8_workspace(args(K=15, lda=15, ldb=15))
    assert need > 0
    refused(-2, lambda: L.cla_q8_mm_dev(args(K=15, lda=15, ldb=15), None))
    refused(-2, lambda: L.cla_q8_mm_dev(args(K=15, lda=15, ldb=15, work=P, workBytes=need - 1), None))
    refused(-2, lambda: L.cla_q8_mm_dev(args(K=15, lda=15, ldb=15, work=P + 16, workBytes=need), None))
    refused(-2, lambda: L.cla_q8_mm_dev(None, None))
    for code, kw in ((-3, {"type": 4}), (-2, {"by": 2}), (-4, {"ldx": 3}), (-4, {"ldq": 3}), (-2, {"q": None}), (-2, {"scale": None})):
        v = {"type": 1, "by": 0, "ldx": 8, "ldq": 8, "q": P, "scale": P, **kw}
        refused(code, lambda: L.cla_q8_quantize_dev(v["type"], P, v["ldx"], 4, 8, v["by"], v["q"], v["ldq"], v["scale"], 0, None))


def test_gated_refusals():
    L = native.lib()

    def args(**kw):
        c = native.cla_gated(M=4, D=8, F=16, x=P, wg=P, wu=P, ldx=8, ldwg=16, ldwu=16, h=P, g=P, u=P, ldh=16, ldg=16, ldu=16, dh=P, lddh=16, dx=P,
                             dwg=P, dwu=P, lddx=8, lddwg=16, lddwu=16, work=P, workBytes=1 << 20, type=2, act=0, wTrans=0, device=0)
        for k, v in kw.items():
            if k == "p":
                c.drop.p = v
            else:
                setattr(c, k, v)
        return C.byref(c)

    both = ((-3, {"type": 1}), (-3, {"act": 5}), (-3, {"act": -1}), (-2, {"wTrans": 2}), (-4, {"D": -1}), (-4, {"ldx": 7}), (-4, {"ldwg": 15}),
            (-4, {"wTrans": 1, "ldwg": 7}), (-2, {"wu": None}), (-2, {"x": None}), (-2, {"p": 1.0}), (-4, {"ldg": 15}), (-2, {"u": P + 1}))
    for code, kw in both + ((-2, {"h": None}), (-4, {"ldh": 15}), (-2, {"g": None})):
        refused(code, lambda: L.cla_gated_fwd_dev(args(**kw), None))
        refused(code, lambda: L.cla_gated_workspace(args(**kw), 0))
    for code, kw in both + ((-2, {"dh": None}), (-4, {"lddh": 15}), (-2, {"g": None}), (-2, {"dwu": None}), (-4, {"lddx": 7}), (-4, {"lddwu": 15}),
                            (-2, {"workBytes": 16}), (-2, {"work": None}), (-2, {"work": P + 8})):
        refused(code, lambda: L.cla_gated_bwd_dev(args(**kw), None))
    assert L.cla_gated_workspace(args(), 0) == 0
    assert L.cla_gated_workspace(args(), 1) >= 2 * 4 * 16 * 2


def test_rows_of_a_block_refusals():
    L = native.lib()
    h = check(L.cla_create(10, 2, 0))
    for f in (lambda: L.cla_rows_workspace(h, 4, 1), lambda: L.cla_q8_rmm_workspace(h, 4),
              lambda: L.cla_decompress_rows_dev(h, 0, 4, 1, P, 2, P, 1 << 20, None),
              lambda: L.cla_q8_rmm_dev(h, P, 16, P, 4, 1, P, 4, P, 1 << 20, None)):
        refused(-6, f)  # cla_finalize comes first
    check(L.cla_destroy(h))
    refused(-1, lambda: L.cla_rows_workspace(h, 4, 1))


def test_classes_refuse_host_tensors():
    x, q, s = torch.ones(4, 8), torch.ones(4, 8, dtype=torch.int8), torch.ones(4)
    for f in (lambda: CLALibDropout.apply(x, 0.5, 1), lambda: CLALibQ8.quantizeRows(x), lambda: CLALibQ8.quantizeCols(x),
              lambda: CLALibQ8.matrixMult(q, s, q, s), lambda: CLALibQ8.linear(x, q, s),
              lambda: CLALibGated.forward(x.half(), x.t().half(), x.t().half())):
        refused(-2, f)
    refused(-3, lambda: CLALibQ8.matrixMult(x, s, q, s))
