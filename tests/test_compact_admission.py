"""iomb_cache_compact refuses keys and values with planes in common, also where both are views of
one owner (no GPU needed: refused before any device work)."""
import ctypes

import pytest

from iom_b200 import _abi
from iom_b200.tensor import DataType, TensorSpec, TensorView
from support import HostTensor

WORD = 0x10000          # never dereferenced


@pytest.mark.parametrize("k,v", [
    ((0, 2, 1), (0, 2, 1)), ((0, 4, 1), (1, 4, 1)), ((0, 4, 1), (4, 4, 1)), ((3, 4, 1), (0, 4, 1)), ((0, 2, 1), (5, 2, 1)),
    ((0, 4, 1), (2, 3, 1)), ((0, 1, 1), (10, 2, 1)), ((10, 2, 1), (0, 1, 1)),
])
def test_planes_in_common(k, v):
    owner = HostTensor((20, 40, 64), DataType.BF16)
    spec = TensorSpec((3, 2, 40, 64), DataType.BF16)
    views = [TensorView(owner, spec, at[0], at[1:]).as_abi() for at in (k, v)]
    assert _abi.load_library().iomb_cache_compact(ctypes.byref(views[0]), ctypes.byref(views[1]), WORD, WORD, 4, WORD, WORD,
                                                  None) == 1
    assert "overlap" in _abi.last_error()
