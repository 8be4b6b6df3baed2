"""B200-native compressed linear algebra for SystemDS column groups (matrix-multiply path)."""
from .cmb import (CHAIN_XtXv, CHAIN_XtwXv, CLALibDecompress, CLALibLeftMultBy, CLALibMatrixMult, CLALibMMChain,
                  CLALibRightMultBy,
                  CLALibTSMM, CompressedMatrixBlock)
from .native import CLAError

__all__ = ["CompressedMatrixBlock", "CLALibRightMultBy", "CLALibLeftMultBy", "CLALibTSMM", "CLALibMMChain",
           "CLALibDecompress", "CLALibMatrixMult", "CLALibQ8", "CLALibGated", "CLALibDropout", "CLAError", "CHAIN_XtXv", "CHAIN_XtwXv"]


def __getattr__(name):  # (the dense operators take torch tensors: torch is imported when one of them is asked for)
    if name in ("CLALibQ8", "CLALibGated", "CLALibDropout"):
        from . import dense
        return getattr(dense, name)
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
