"""Arguments of csrc/mr_torch.cpp's functions that are no numbers or truth values: the Python error
that they raise, not one about the call itself. No GPU needed."""
import ctypes as C
import os
import subprocess
import sys

import pytest
import torch

from minirun_moe import _lib as L
from minirun_moe import sorted_tokens as S


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


CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(L.__file__))), "csrc")


@pytest.fixture
def reloaded(monkeypatch):
    monkeypatch.setattr(L, "_torch_ext", None)
    return monkeypatch


def takes_nothing(ext):
    ids = torch.zeros((4, 2), dtype=torch.int32)
    return ext.sort(0, 0, ids, 3) is None and ext.quantize(0, 0, ids, False) is None


def test_a_build_without_the_module_has_the_calls_by_ctypes(reloaded, tmp_path):
    reloaded.setattr(L, "TORCH_PATH", str(tmp_path / "none.so"))
    assert takes_nothing(L.load_torch()) and L.load_torch() is L.load_torch()
    mem = torch.arange(2 * 8 + 4, dtype=torch.int32)
    p = S.SortedTokens._of(mem, 4, 2, 3)
    assert p.order.tolist() == list(range(8)) and p.offsets.tolist() == list(range(16, 20))
    assert p.inverse.tolist() == [[8, 9], [10, 11], [12, 13], [14, 15]]


def test_a_module_that_does_not_load_warns(reloaded, tmp_path):
    bad = tmp_path / "bad.so"
    bad.write_bytes(b"no library")
    reloaded.setattr(L, "TORCH_PATH", str(bad))
    with pytest.warns(UserWarning, match="is not used"):
        assert takes_nothing(L.load_torch())


def test_a_module_for_another_torch_is_not_used(reloaded):
    reloaded.setattr(torch, "__version__", "1.0.0")
    with pytest.warns(UserWarning, match="this is 1.0.0"):
        assert takes_nothing(L.load_torch())


def test_the_makefile_needs_no_torch():
    def plan(python):
        return subprocess.run(["make", "-n", "-B", "-C", CSRC, f"PYTHON={python}"], check=True,
                              capture_output=True, text=True).stdout

    assert "mr_torch.cpp" in plan(sys.executable)
    without = plan("false")
    assert "mr_torch.cpp" not in without and "libminirun_moe.so" in without
