"""Refusals of the token-sorting and 4-bit entry points that need no GPU: every
check that precedes the first CUDA call, through the C ABI with a context
pointer that is never used and through the Python functions on CPU tensors."""
import ctypes as C

import pytest
import torch

import minirun_moe as M
from minirun_moe import _lib as L


def test_null_context_is_refused():
    lib = L.load()
    s = L.mr_sorted(16, 16, 16, 4, 2, 3)
    d = L.mr_mxfp4_desc(16, 16, 0, 8, 64)
    calls = [
        lambda: lib.mr_moe_sort(None, 16, 4, 2, 3, 16, 16, 16, None),
        lambda: lib.mr_moe_dispatch(None, 16, 0, 64, 64, C.byref(s), 16, None),
        lambda: lib.mr_moe_dispatch_backward(None, 16, 0, 64, 64, C.byref(s), 16, None),
        lambda: lib.mr_moe_combine(None, 16, 0, 64, 64, 16, None, C.byref(s), 16, None),
        lambda: lib.mr_moe_combine_backward(None, 16, 64, 16, 64, 0, 64, 16, C.byref(s), 16, 16,
                                            None),
        lambda: lib.mr_mxfp4_quantize(None, 16, 0, 4, 64, 64, 16, 16, None, None),
        lambda: lib.mr_mxfp4_quantize_swiglu(None, 16, 0, 4, 64, 128, 0.0, 16, 16, None),
        lambda: lib.mr_mxfp4_scaled_mm(None, C.byref(d), C.byref(d), 0, 16, None),
        lambda: lib.mr_mxfp4_grouped_mm(None, C.byref(d), C.byref(d), C.byref(s), 0, 0, 16, None),
    ]
    for f in calls:
        assert f() == L.MR_ERR_INVALID_ARGUMENT


def test_cpu_tensors_are_refused():
    ids = torch.zeros((4, 2), dtype=torch.int32)
    with pytest.raises(M.AffineBridgeError):
        M.moe_sort(ids, 3)
    with pytest.raises(M.AffineBridgeError, match="CUDA int32"):
        M.SortedTokens(torch.zeros(8, dtype=torch.int32), ids, torch.zeros(4, dtype=torch.int32),
                       3)
    with pytest.raises(M.MXFP4BridgeError, match="must be a CUDA"):
        M.mxfp4_quantize(torch.zeros((2, 64)))
    with pytest.raises(M.MXFP4BridgeError, match="must be a CUDA"):
        M.mxfp4_quantize_swiglu(torch.zeros((2, 64)))
    w = M.MXFP4Weights(torch.zeros((8, 8), dtype=torch.int32),
                       torch.zeros((8, 2), dtype=torch.uint8))
    with pytest.raises(M.MXFP4BridgeError, match="one CUDA device"):
        M.mxfp4_scaled_mm(w, w)


def test_sorted_struct_matches_the_c_compiler(tmp_path):
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = [f[0] for f in L.mr_sorted._fields_]
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "minirun_moe.h"\n'
                   'int main(void) { printf("%zu", sizeof(mr_sorted));\n' +
                   "".join(f'printf(" %zu", offsetof(mr_sorted, {n}));\n' for n in names) +
                   "return 0; }\n")
    exe = tmp_path / "s"
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", str(exe)],
                   check=True)
    got = list(map(int, subprocess.check_output([str(exe)]).split()))
    assert got == [C.sizeof(L.mr_sorted)] + [getattr(L.mr_sorted, n).offset for n in names]


def test_short_way_takes_only_the_plain_case():
    """csrc/mr_torch.cpp answers None for what it leaves to the Python functions: CPU tensors,
    other types, a wrong number of arguments."""
    ext = L.load_torch()
    ids = torch.zeros((4, 2), dtype=torch.int32)
    x = torch.zeros((4, 64))
    plan = L.mr_sorted(16, 16, 16, 4, 2, 3)
    at = C.addressof(plan)
    w = torch.zeros((4, 2))
    p, s = torch.zeros((4, 8), dtype=torch.int32), torch.zeros((4, 2), dtype=torch.uint8)
    assert ext.sort(0, 0, ids, 3) is None
    assert ext.sort(0, 0, ids) is None
    assert ext.sort(0, 0, "ids", 3) is None
    assert ext.dispatch(0, 0, x, at) is None
    assert ext.dispatch_backward(0, 0, x, at) is None
    assert ext.combine(0, 0, x, w, at) is None
    assert ext.combine_backward(0, 0, x, x, w, at) is None
    assert ext.quantize(0, 0, x, False) is None
    assert ext.quantize_swiglu(0, 0, x, 0.0) is None
    assert ext.scaled_mm(0, 0, p, s, p, s, False) is None
    assert ext.grouped_mm(0, 0, p, s, p, s, False, at, False) is None
    with pytest.raises(TypeError):
        ext.bind(1, 2)


def test_short_way_binds_every_function_in_order():
    import os
    import re
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = open(os.path.join(root, "minirun-app_b200", "csrc", "mr_torch.cpp")).read()
    names = re.findall(r"decltype\(&(mr_\w+)\)", src)
    assert tuple(names) == L._TORCH_API
