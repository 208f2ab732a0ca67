"""Arguments of csrc/mr_torch.cpp's functions that are no numbers or truth values: the Python error
that they raise, not one about the call itself. No GPU needed."""
import ctypes as C

import pytest
import torch

from minirun_moe import _lib as L


def test_a_wrong_number_raises_its_own_error():
    ext = L.load_torch()
    ids = torch.zeros((4, 2), dtype=torch.int32)
    plan = L.mr_sorted(16, 16, 16, 4, 2, 3)
    with pytest.raises(TypeError):
        ext.sort(0, 0, ids, 3.0)
    with pytest.raises(OverflowError):
        ext.sort(0, 0, ids, 2 ** 70)
    assert ext.sort(0, 0, ids, -1) is None
    with pytest.raises(TypeError):
        ext.views(torch.zeros(20, dtype=torch.int32), 4, "2", 3)
    with pytest.raises(TypeError):
        ext.dispatch(0, None, torch.zeros((4, 64)), C.addressof(plan))
    with pytest.raises(TypeError):
        ext.quantize_swiglu(0, 0.5, torch.zeros((4, 64)), 0.0)
