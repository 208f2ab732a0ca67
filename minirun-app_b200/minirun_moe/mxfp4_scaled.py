"""4 bits on both sides: quantisation to MXFP4 and MXFP4 x MXFP4 products,
over libminirun_moe's C ABI.

Activations take the form of the weights: ``MXFP4Weights`` of ``[rows, in]``
(``out_features`` counts the rows). ``mxfp4_quantize`` makes either from bf16,
f16 or fp32 tensors; the products run on the tensor cores' block-scaled 4-bit
form (exact products and scales, fp32 sums), one matrix
(``mxfp4_scaled_mm``) or an expert stack over rows sorted by expert
(``mxfp4_grouped_mm``).
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib as L
from .bridge import Context, _raw_stream
from .mxfp4 import MXFP4BridgeError, MXFP4Weights
from .sorted_tokens import SortedTokens

_IN_DTYPES = {torch.bfloat16: L.MR_DTYPE_BF16, torch.float16: L.MR_DTYPE_F16,
              torch.float32: L.MR_DTYPE_F32}
_OUT_DTYPES = {torch.bfloat16: L.MR_DTYPE_BF16, torch.float32: L.MR_DTYPE_F32}


def _checked(name: str, x: torch.Tensor):
    """(x, its shape, row stride) for rows that the quantiser reads in place: the last axis
    contiguous, the rows one stride apart; otherwise of a copy."""
    shape = x.shape
    if len(shape) not in (2, 3) or not x.is_cuda or x.dtype not in _IN_DTYPES:
        raise MXFP4BridgeError(
            f"{name} must be a CUDA bfloat16, float16 or float32 [rows, inFeatures] or [experts, "
            f"rows, inFeatures] tensor, got {list(shape)} {x.dtype} on {x.device}")
    n = shape[-1]
    if x.is_contiguous():
        return x, shape, n
    if len(shape) == 2 and x.stride(1) == 1 and (shape[0] <= 1 or x.stride(0) >= n):
        return x, shape, max(x.stride(0), n)
    return x.contiguous(), shape, n


def _weights_of(packed: torch.Tensor, scales: torch.Tensor, rows: int, width: int,
                experts: int | None) -> MXFP4Weights:
    w = MXFP4Weights.__new__(MXFP4Weights)  # shapes and types are right by construction
    w.packed, w.scales = packed, scales
    w.experts, w.out_features, w.in_features = experts, rows, width
    w._keepalive = None
    return w


def mxfp4_quantize(x: torch.Tensor, values: bool = False):
    """``x`` [rows, in] or [experts, rows, in] in MXFP4 (see mr_mxfp4_quantize for the rounding).
    With ``values`` the pair (codes, values): the numbers the codes stand for in x's type, what a
    training step with 4-bit forward values multiplies with. No gradient is recorded: how it passes
    the rounding is the caller's choice (straight through: ``x + (values - x.detach())``)."""
    if x.is_cuda and x.dim() == 2:
        ctx = Context.get(x.get_device())
        r = L.load_torch().quantize(ctx.address, ctx.device, x, values)
        if r is not None:
            if r.__class__ is int:
                ctx.check("mr_mxfp4_quantize", r)
            q = _weights_of(r[0], r[1], x.shape[0], x.shape[1], None)
            return (q, r[2]) if values else q
    x, shape, stride = _checked("x", x)
    if len(shape) == 2:
        experts, (rows, width) = None, shape
        lead = (rows,)
    else:
        experts, rows, width = shape
        lead = (experts, rows)
    if width % 32 != 0 or width == 0:
        raise MXFP4BridgeError(
            f"inFeatures {width} is not a multiple of groupSize 32; partial final groups are "
            "not supported")
    dev = x.device
    packed = x.new_empty((*lead, width // 8), dtype=torch.int32)
    scales = x.new_empty((*lead, width // 32), dtype=torch.uint8)
    out = x.new_empty(shape) if values else None
    ctx = Context.get(dev.index)
    st = L.load().mr_mxfp4_quantize(
        ctx.handle, x.data_ptr(), _IN_DTYPES[x.dtype], rows if experts is None else rows * experts,
        width, stride, packed.data_ptr(), scales.data_ptr(),
        None if out is None else out.data_ptr(), _raw_stream(dev))
    if st:
        ctx.check("mr_mxfp4_quantize", st)
    q = _weights_of(packed, scales, rows, width, experts)
    return (q, out) if values else q


def mxfp4_quantize_swiglu(gate_up: torch.Tensor, limit: float = 0.0) -> MXFP4Weights:
    """``silu(gate) * up`` of rows ``[gate | up]`` in MXFP4, [rows, in]; ``limit`` > 0 clamps
    ``gate <= limit`` and ``-limit <= up <= limit`` first."""
    if gate_up.is_cuda and gate_up.dim() == 2:
        ctx = Context.get(gate_up.get_device())
        r = L.load_torch().quantize_swiglu(ctx.address, ctx.device, gate_up, limit)
        if r is not None:
            if r.__class__ is int:
                ctx.check("mr_mxfp4_quantize_swiglu", r)
            return _weights_of(r[0], r[1], gate_up.shape[0], gate_up.shape[1] // 2, None)
    x, shape, stride = _checked("gate_up", gate_up)
    if len(shape) != 2 or shape[1] % 64 != 0 or shape[1] == 0:
        raise MXFP4BridgeError(
            f"gate_up must be [rows, 2 * inter] with inter a multiple of 32, got {list(shape)}")
    rows, width = shape[0], shape[1] // 2
    dev = x.device
    packed = x.new_empty((rows, width // 8), dtype=torch.int32)
    scales = x.new_empty((rows, width // 32), dtype=torch.uint8)
    ctx = Context.get(dev.index)
    st = L.load().mr_mxfp4_quantize_swiglu(
        ctx.handle, x.data_ptr(), _IN_DTYPES[x.dtype], rows, width, stride, limit,
        packed.data_ptr(), scales.data_ptr(), _raw_stream(dev))
    if st:
        ctx.check("mr_mxfp4_quantize_swiglu", st)
    return _weights_of(packed, scales, rows, width, None)


def _operands(a: MXFP4Weights, w: MXFP4Weights, out_dtype: torch.dtype) -> int:
    if a.experts is not None:
        raise MXFP4BridgeError("activations are a single [rows, inFeatures] matrix, not a stack")
    if a.in_features != w.in_features:
        raise MXFP4BridgeError(f"a has {a.in_features} features, weights expect {w.in_features}")
    if not a.packed.is_cuda or a.packed.device != w.packed.device:
        raise MXFP4BridgeError(
            f"a and w must be on one CUDA device, got {a.packed.device} and {w.packed.device}")
    if out_dtype not in _OUT_DTYPES:
        raise MXFP4BridgeError(f"out_dtype must be bfloat16 or float32, got {out_dtype}")
    return _OUT_DTYPES[out_dtype]


def mxfp4_scaled_mm(a: MXFP4Weights, w: MXFP4Weights,
                    out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``a . w^T`` [rows, out] of two MXFP4 matrices, fp32 sums."""
    if a.experts is None and w.experts is None and out_dtype in _OUT_DTYPES and a.packed.is_cuda:
        ctx = Context.get(a.packed.get_device())
        out = L.load_torch().scaled_mm(ctx.address, ctx.device, a.packed, a.scales, w.packed,
                                       w.scales, out_dtype is torch.float32)
        if out is not None:
            if out.__class__ is int:
                ctx.check("mr_mxfp4_scaled_mm", out)
            return out
    dt = _operands(a, w, out_dtype)
    if w.experts is not None:
        raise MXFP4BridgeError("mxfp4_scaled_mm needs a single matrix; use mxfp4_grouped_mm")
    dev = a.packed.device
    out = a.packed.new_empty((a.out_features, w.out_features), dtype=out_dtype)
    ctx = Context.get(dev.index)
    st = L.load().mr_mxfp4_scaled_mm(ctx.handle, C.byref(a.desc()), C.byref(w.desc()), dt,
                                     out.data_ptr(), _raw_stream(dev))
    if st:
        ctx.check("mr_mxfp4_scaled_mm", st)
    return out


def mxfp4_grouped_mm(a: MXFP4Weights, w: MXFP4Weights, plan: SortedTokens,
                     by_token: bool = False,
                     out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``out[r] = w[e] . a[r]`` for the sorted rows r of expert e; zeros in rows without a pair.

    ``a`` holds the sorted rows, or with ``by_token`` the tokens' rows: row r then takes
    ``a[order[r] // top_k]``, read in place, so a token is quantised once whatever top_k is."""
    if a.experts is None and w.experts is not None and out_dtype in _OUT_DTYPES:
        ctx = Context.get(plan.index)
        out = L.load_torch().grouped_mm(ctx.address, plan.index, a.packed, a.scales, w.packed,
                                        w.scales, out_dtype is torch.float32, plan._at, by_token)
        if out is not None:
            if out.__class__ is int:
                ctx.check("mr_mxfp4_grouped_mm", out)
            return out
    dt = _operands(a, w, out_dtype)
    if w.experts is None:
        raise MXFP4BridgeError("mxfp4_grouped_mm needs an expert stack; use mxfp4_scaled_mm")
    if w.experts != plan.experts:
        raise MXFP4BridgeError(
            f"the stack has {w.experts} experts, the tokens are sorted into {plan.experts}")
    want = plan.tokens if by_token else plan.rows
    if a.out_features != want:
        raise MXFP4BridgeError(
            f"a must have {want} rows ({'tokens' if by_token else 'sorted rows'}), got "
            f"{a.out_features}")
    dev = a.packed.device
    if plan.device != dev:
        raise MXFP4BridgeError(f"a is on {dev}, the sorted tokens on {plan.device}")
    out = a.packed.new_empty((plan.rows, w.out_features), dtype=out_dtype)
    ctx = Context.get(dev.index)
    st = L.load().mr_mxfp4_grouped_mm(ctx.handle, C.byref(a.desc()), C.byref(w.desc()), plan._ref,
                                      int(by_token), dt, out.data_ptr(), _raw_stream(dev))
    if st:
        ctx.check("mr_mxfp4_grouped_mm", st)
    return out
