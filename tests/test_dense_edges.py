"""What the dense operators refuse on the host, beyond test_dense.py, and how they are imported."""
import ctypes as C
import os
import re
import subprocess
import sys

import pytest
import torch

from systemds_b200 import CLAError, CLALibDecompress, CLALibQ8, CompressedMatrixBlock, native
from systemds_b200.dense import _drop, _type
from systemds_b200.native import check

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
M, K, N = 6, 48, 48
A, B, SA, SB, OUT, WORK, MORE = ((i + 1) << 24 for i in range(7))  # addresses that nothing reads: the calls below are refused on the host


def refused(code, f):
    with pytest.raises(CLAError) as e:
        check(f())
    assert e.value.code == code, str(e.value)


def test_8_bit_products_onto_their_operands():
    L = native.lib()

    def mm(**kw):
        c = native.cla_q8(M=M, N=N, K=K, a=A, lda=K, aScale=SA, b=B, ldb=K, bScale=SB, out=OUT, ldo=N, work=WORK, workBytes=1 << 20, aType=4, outType=1, device=0)
        for k, v in kw.items():
            setattr(c, k, v)
        return L.cla_q8_mm_dev(C.byref(c), None)

    for at in (A, A + 4, A + (M - 1) * K, A - (M - 1) * N * 4, B, B + N * K - 4, SA, SA + 4 * M - 4, SB, SB + 4 * N - 4):
        refused(-2, lambda: mm(out=at))
    refused(-2, lambda: mm(lda=240, ldo=60, out=A + 40))  # (240 bytes a row each, side by side but for 8 bytes)
    refused(-2, lambda: mm(lda=401, ldo=50, out=A + 48 + 12))  # (the rows' distances differ: they meet in some later row)
    refused(-2, lambda: mm(b=B + 1, work=B))  # (copied to the workspace, off its boundary)
    refused(-2, lambda: mm(b=B + 1, work=OUT))
    for at in (A, A + 16):
        refused(-2, lambda: L.cla_q8_quantize_dev(1, A, 8, 4, 8, 0, at, 8, SA, 0, None))
        refused(-2, lambda: L.cla_q8_quantize_dev(1, A, 8, 4, 8, 1, OUT, 8, at, 0, None))
    refused(-2, lambda: L.cla_q8_quantize_dev(1, A, 8, 4, 8, 0, OUT, 8, OUT + 12, 0, None))


def test_gated_blocks_onto_their_operands():
    L = native.lib()

    def call(backward, **kw):
        c = native.cla_gated(M=M, D=K, F=K, x=A, wg=B, wu=SA, ldx=K, ldwg=K, ldwu=K, h=OUT, g=MORE, u=MORE << 1, ldh=K, ldg=K, ldu=K, dh=SB, lddh=K,
                             dx=OUT, dwg=OUT << 1, dwu=OUT << 2, lddx=K, lddwg=K, lddwu=K, work=WORK, workBytes=1 << 20, type=2, act=0, wTrans=0, device=0)
        for k, v in kw.items():
            setattr(c, k, v)
        return (L.cla_gated_bwd_dev if backward else L.cla_gated_fwd_dev)(C.byref(c), None)

    last = 2 * (M * K - 1)
    for kw in ({"h": A}, {"h": A + last}, {"h": B}, {"h": SA + 2 * (K * K - 1)}, {"g": A}, {"u": B}, {"h": MORE}, {"u": MORE + 2}):
        refused(-2, lambda: call(False, **kw))
    for kw in ({"dx": A}, {"dx": SB + last}, {"dx": MORE}, {"dwg": B}, {"dwu": SA}, {"dwg": MORE << 1}, {"dwu": OUT << 1}, {"work": A}, {"work": OUT}):
        refused(-2, lambda: call(True, **kw))


def test_dropout_partly_onto_its_operand():
    L = native.lib()

    def call(x, ldx, y, ldy, rows=4, cols=8):
        return L.cla_dropout_dev(1, x, ldx, rows, cols, y, ldy, C.byref(native.cla_drop(0.5, 1, 2, 0)), 0, None)

    for at in (A + 4, A + 32, A + 96 + 28, A - 4, A - 96 - 28):
        refused(-2, lambda: call(A, 8, at, 8))
    refused(-2, lambda: call(A, 8, A, 16))
    refused(-2, lambda: call(A, 20, A + 28, 20))
    refused(-2, lambda: call(A, 20, A + 32, 21, rows=8))  # (the sixth row has moved on to the next one's place)


def test_rows_whose_end_leaves_64_bits():
    L = native.lib()
    for row0 in ((1 << 63) - 1, (1 << 63) - 4, (1 << 63) - 6):
        d = native.cla_drop(0.5, 1, 2, row0)
        refused(-2, lambda: L.cla_dropout_dev(1, A, 8, M, 8, B, 8, C.byref(d), 0, None))
        c = native.cla_gated(M=M, D=K, F=K, x=A, wg=B, wu=SA, ldx=K, ldwg=K, ldwu=K, h=OUT, ldh=K, drop=d, type=2)
        refused(-2, lambda: L.cla_gated_fwd_dev(C.byref(c), None))
        refused(-2, lambda: L.cla_gated_workspace(C.byref(c), 0))


def test_arguments_of_other_kinds():
    """Failures are CLAError also where an argument is nothing that the call knows."""
    for args in ((None, 1, 0, 0), ("0.5", "1", 0, 0), (0.5, 1.5, 0, 0), (0.5, "1", 0, 0), (0.5, 1, None, 0), (0.5, 1, 0, [0]), (0.5, -1, 0, 0), (0.5, 1, 1 << 64, 0)):
        refused(-2, lambda: _drop(*args))
    d = _drop(torch.tensor(0.5), torch.tensor(3), torch.tensor(1 << 40), torch.tensor(7))
    assert (d.p, d.seed, d.step, d.row0) == (0.5, 3, 1 << 40, 7)
    for dtype in (torch.int32, "bf16", None, [torch.float32], float):
        refused(-3, lambda: _type(dtype, "type"))
    block, x = CompressedMatrixBlock(4, 2, []), torch.ones(4, 2)
    block._handle = 1  # (refused before anybody asks for it)
    for args in ((x, 0, 2, torch.float32), (block, "0", 2, torch.float32), (block, 0, 1.5, torch.float32), (block, 0, 2, torch.float32, [1]),
                 (block, 0, 2, torch.float32, x[:2].numpy())):
        refused(-2, lambda: CLALibDecompress.rows(*args))
    refused(-3, lambda: CLALibDecompress.rows(block, 0, 2, "bf16"))
    refused(-4, lambda: CLALibDecompress.rows(block, 0, 2, torch.float32, x))
    refused(-2, lambda: CLALibQ8.rightMultByMatrix(x, x, x))
    block._handle = 0


@pytest.mark.parametrize("torch_is_there", [True, False])
def test_star_import(torch_is_there):
    """Without torch the compressed products are imported alone; torch waits until it is asked for."""
    code = ("import sys\n" + ("" if torch_is_there else "sys.modules['torch'] = None\n") + "import systemds_b200\n"
            "assert sys.modules.get('torch') is None\nfrom systemds_b200 import *\nCompressedMatrixBlock, CLALibRightMultBy, CLAError\n"
            f"assert ('CLALibQ8' in globals()) == {torch_is_there}\n"
            "try:\n    from systemds_b200 import CLALibDropout\n    there = True\nexcept ImportError:\n    there = False\n"
            f"assert there == {torch_is_there}\n")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert r.returncode == 0, r.stderr


def test_dense_launchers_share_no_plain_numbers():
    """What threads share and write: atomics, marks of OncePerDevice, or each thread's own."""
    for name in ("cla_dense.cu", "cla_dense.cuh", "cla_gemm.cu"):
        with open(os.path.join(ROOT, "systemds_b200", "csrc", name)) as f:
            found = re.findall(r"\bstatic\s+(?:bool|int|int32_t|int64_t|size_t|unsigned)\s+(\w+)\s*(?:;|=|\[)", f.read())
        assert found == [], name
