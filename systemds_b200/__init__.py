"""B200-native compressed linear algebra for SystemDS column groups (matrix-multiply path)."""
from importlib.util import find_spec

from .cmb import (CHAIN_XtXv, CHAIN_XtwXv, CLALibDecompress, CLALibLeftMultBy, CLALibMatrixMult, CLALibMMChain,
                  CLALibRightMultBy,
                  CLALibTSMM, CompressedMatrixBlock)
from .native import CLAError

__all__ = ["CompressedMatrixBlock", "CLALibRightMultBy", "CLALibLeftMultBy", "CLALibTSMM", "CLALibMMChain",
           "CLALibDecompress", "CLALibMatrixMult", "CLAError", "CHAIN_XtXv", "CHAIN_XtwXv"]
_DENSE = ("CLALibQ8", "CLALibGated", "CLALibDropout")


def _has_torch() -> bool:
    try:
        return find_spec("torch") is not None
    except ValueError:  # (a module of that name without a specification)
        return True


if _has_torch():  # (a star import asks for every name; the compressed products need numpy alone)
    __all__ += _DENSE


def __getattr__(name):  # (the dense operators take torch tensors: torch is imported when one of them is asked for)
    if name in _DENSE:
        from . import dense
        return getattr(dense, name)
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
