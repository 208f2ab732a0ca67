"""Tokens sorted by expert and back, over libminirun_moe's C ABI.

A router chooses ``top_k`` experts a token (``Selection.ids``). ``moe_sort``
orders the (token, slot) pairs by expert, ``moe_dispatch`` copies the tokens'
rows into that order, the experts work on contiguous rows, and
``moe_combine`` brings their rows back, weighted and summed. Both copies have
their gradients, as functions and through torch's autograd: where an input
requires a gradient, ``moe_dispatch`` and ``moe_combine`` record it. (Gradients
of the gradients and forward-mode tangents are not built and raise; the gradient
functions themselves record nothing.)

An id of -1 is a slot without an expert: it takes no expert's row, its sorted
row comes after all experts' and holds zeros, and the combine adds nothing.
"""
from __future__ import annotations

import ctypes as C

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib as L
from .bridge import AffineBridgeError, Context, _raw_stream

_ROW_DTYPES = {torch.bfloat16: L.MR_DTYPE_BF16, torch.float16: L.MR_DTYPE_F16,
               torch.float32: L.MR_DTYPE_F32}


class SortedTokens:
    """What ``moe_sort`` returns: ``order`` [tokens * top_k] (the pair
    ``token * top_k + slot`` at each sorted row, -1 past the last expert's),
    ``inverse`` [tokens, top_k] (the row of each pair, -1 without an expert)
    and ``offsets`` [experts + 1] (first row of each expert), int32."""

    def __init__(self, order: torch.Tensor, inverse: torch.Tensor, offsets: torch.Tensor,
                 experts: int):
        if inverse.dim() != 2 or order.shape != (inverse.numel(),):
            raise AffineBridgeError(
                f"inverse must be [tokens, top_k] and order [tokens * top_k], got "
                f"{list(inverse.shape)} and {list(order.shape)}")
        if offsets.shape != (experts + 1,):
            raise AffineBridgeError(
                f"offsets must be [{experts + 1}] for {experts} experts, got "
                f"{list(offsets.shape)}")
        for t in (order, inverse, offsets):
            if t.dtype != torch.int32 or not t.is_contiguous() or not t.is_cuda:
                raise AffineBridgeError("sorted tokens are contiguous CUDA int32 tensors")
            if t.device != order.device:
                raise AffineBridgeError("sorted tokens must be on one device")
        self._mem, self._views = None, (order, inverse, offsets)
        self._fill(order.data_ptr(), inverse.data_ptr(), offsets.data_ptr(), inverse.shape[0],
                   inverse.shape[1], experts, order.device)

    def _fill(self, order, inverse, offsets, tokens, top_k, experts, device):
        self.tokens, self.top_k, self.experts = tokens, top_k, experts
        self.rows = tokens * top_k
        self.device, self.index = device, device.index
        self._c = L.mr_sorted(order, inverse, offsets, tokens, top_k, experts)
        self._ref, self._at = C.byref(self._c), C.addressof(self._c)

    @classmethod
    def _of(cls, mem: torch.Tensor, tokens: int, top_k: int, experts: int) -> "SortedTokens":
        """The plan in one buffer (order, inverse, offsets); its views are made when asked for."""
        s = cls.__new__(cls)
        s._mem, s._views = mem, None
        at, P = mem.data_ptr(), 4 * tokens * top_k
        s._fill(at, at + P, at + 2 * P, tokens, top_k, experts, mem.device)
        return s

    def _split(self):
        if self._views is None:
            P, E = self.rows, self.experts
            self._views = L.load_torch().views(self._mem, self.tokens, self.top_k, E) or (
                self._mem[:P], self._mem[P:2 * P].view(self.tokens, self.top_k),
                self._mem[2 * P:2 * P + E + 1])
        return self._views

    def _version(self) -> tuple:
        """Tells whether the plan's tensors were written between two calls (in place, by torch; an
        inference tensor does not count its writes)."""
        mine = self._views if self._mem is None else (self._mem,)
        return tuple(-1 if t.is_inference() else t._version for t in mine)

    @property
    def order(self) -> torch.Tensor:
        return self._split()[0]

    @property
    def inverse(self) -> torch.Tensor:
        return self._split()[1]

    @property
    def offsets(self) -> torch.Tensor:
        return self._split()[2]


def moe_sort(ids: torch.Tensor, experts: int) -> SortedTokens:
    """The pairs of ``ids`` [tokens, top_k] in the order of their experts, stable."""
    if ids.is_cuda and ids.dim() == 2:
        ctx = Context.get(ids.get_device())
        mem = L.load_torch().sort(ctx.address, ctx.device, ids, experts)
        if mem is not None:
            if mem.__class__ is int:
                ctx.check("mr_moe_sort", mem)
            T, k = ids.shape
            return SortedTokens._of(mem, T, k, experts)
    if ids.dim() != 2 or not ids.is_cuda:
        raise AffineBridgeError("ids must be a CUDA [tokens, top_k] tensor")
    if ids.dtype != torch.int32:
        if ids.dtype != torch.int64:
            raise AffineBridgeError(f"ids must be int32 or int64, got {ids.dtype}")
        # an id out of int32's range stays out of range, and -1 the only one without an error
        ids = ids.clamp(-2, 2 ** 31 - 1).to(torch.int32)
    if not ids.is_contiguous():
        ids = ids.contiguous()
    if not -2 ** 31 <= experts < 2 ** 31:
        raise AffineBridgeError(f"experts must be a number of 32 bits, got {experts}")
    T, k = ids.shape
    mem = ids.new_empty((2 * T * k + min(max(experts, 0), 1024) + 1,))  # more are refused
    s = SortedTokens._of(mem, T, k, experts)
    c, ctx = s._c, Context.get(s.device.index)
    st = L.load().mr_moe_sort(ctx.handle, ids.data_ptr(), T, k, experts, c.order, c.inverse,
                              c.offsets, _raw_stream(s.device))
    if st:
        ctx.check("mr_moe_sort", st)
    return s


def _rows(name: str, t: torch.Tensor, rows: int, plan: SortedTokens):
    """(rows with a contiguous last axis, hidden, row stride) of a [rows, hidden] tensor of a
    supported type on the plan's device."""
    shape = t.shape
    if len(shape) != 2 or shape[0] != rows:
        raise AffineBridgeError(f"{name} must be [{rows}, hidden], got {list(shape)}")
    if t.dtype not in _ROW_DTYPES:
        raise AffineBridgeError(f"{name} must be bfloat16, float16 or float32, got {t.dtype}")
    if t.device != plan.device:
        raise AffineBridgeError(f"{name} is on {t.device}, the sorted tokens on {plan.device}")
    H = shape[1]
    if t.is_contiguous():
        return t, H, H
    if t.stride(1) != 1 or (rows > 1 and t.stride(0) < H):
        return t.contiguous(), H, H
    return t, H, max(t.stride(0), H)


def _weights(w: torch.Tensor, plan: SortedTokens) -> torch.Tensor:
    if w.shape != (plan.tokens, plan.top_k) or w.dtype != torch.float32 or (
            w.device != plan.device):
        raise AffineBridgeError(
            f"weights must be [{plan.tokens}, {plan.top_k}] float32 on {plan.device}, got "
            f"{list(w.shape)} {w.dtype} on {w.device}")
    return w if w.is_contiguous() else w.contiguous()


def _fast(name: str, plan: SortedTokens, *args):
    """The call by its short way, or None where the tensors are not the plain case."""
    ctx = Context.get(plan.index)
    r = getattr(L.load_torch(), name)(ctx.address, plan.index, *args, plan._at)
    if r.__class__ is int:
        ctx.check("mr_moe_" + name, r)
    return r


def _dispatch(x: torch.Tensor, plan: SortedTokens) -> torch.Tensor:
    xs = _fast("dispatch", plan, x)
    if xs is not None:
        return xs
    x, H, stride = _rows("x", x, plan.tokens, plan)
    xs = x.new_empty((plan.rows, H))
    ctx = Context.get(plan.device.index)
    st = L.load().mr_moe_dispatch(ctx.handle, x.data_ptr(), _ROW_DTYPES[x.dtype], stride, H,
                                  plan._ref, xs.data_ptr(), _raw_stream(plan.device))
    if st:
        ctx.check("mr_moe_dispatch", st)
    return xs


def moe_dispatch_backward(dxs: torch.Tensor, plan: SortedTokens) -> torch.Tensor:
    """Gradient of ``moe_dispatch``: ``dx[t] = sum_j dxs[inverse[t, j]]``, fp32 sums."""
    dx = _fast("dispatch_backward", plan, dxs)
    if dx is not None:
        return dx
    dxs, H, stride = _rows("dxs", dxs, plan.rows, plan)
    dx = dxs.new_empty((plan.tokens, H))
    ctx = Context.get(plan.device.index)
    st = L.load().mr_moe_dispatch_backward(ctx.handle, dxs.data_ptr(), _ROW_DTYPES[dxs.dtype],
                                           stride, H, plan._ref, dx.data_ptr(),
                                           _raw_stream(plan.device))
    if st:
        ctx.check("mr_moe_dispatch_backward", st)
    return dx


def _combine(ys, weights, plan, base) -> torch.Tensor:
    if base is None:
        out = _fast("combine", plan, ys, weights)
        if out is not None:
            return out
    ys, H, stride = _rows("ys", ys, plan.rows, plan)
    weights = _weights(weights, plan)
    at = None
    if base is not None:
        if base.shape != (plan.tokens, H) or base.dtype != ys.dtype or base.device != ys.device:
            raise AffineBridgeError(
                f"base must be [{plan.tokens}, {H}] {ys.dtype} on {ys.device}, got "
                f"{list(base.shape)} {base.dtype} on {base.device}")
        base = base.contiguous()
        at = base.data_ptr()
    out = ys.new_empty((plan.tokens, H))
    ctx = Context.get(plan.device.index)
    st = L.load().mr_moe_combine(ctx.handle, ys.data_ptr(), _ROW_DTYPES[ys.dtype], stride, H,
                                 weights.data_ptr(), at, plan._ref, out.data_ptr(),
                                 _raw_stream(plan.device))
    if st:
        ctx.check("mr_moe_combine", st)
    return out


def moe_combine_backward(dout: torch.Tensor, ys: torch.Tensor, weights: torch.Tensor,
                         plan: SortedTokens) -> tuple[torch.Tensor, torch.Tensor]:
    """Gradients ``(dys, dweights)`` of ``moe_combine``; that of ``base`` is ``dout``."""
    both = _fast("combine_backward", plan, dout, ys, weights)
    if both is not None:
        return both
    ys, H, stride = _rows("ys", ys, plan.rows, plan)
    dout, Hd, dstride = _rows("dout", dout, plan.tokens, plan)
    if dout.dtype != ys.dtype or Hd != H:
        raise AffineBridgeError(
            f"dout must be [{plan.tokens}, {H}] {ys.dtype}, got {list(dout.shape)} {dout.dtype}")
    weights = _weights(weights, plan)
    dys = ys.new_empty((plan.rows, H))
    dw = weights.new_empty((plan.tokens, plan.top_k))
    ctx = Context.get(plan.device.index)
    st = L.load().mr_moe_combine_backward(
        ctx.handle, dout.data_ptr(), dstride, ys.data_ptr(), stride, _ROW_DTYPES[ys.dtype], H,
        weights.data_ptr(), plan._ref, dys.data_ptr(), dw.data_ptr(), _raw_stream(plan.device))
    if st:
        ctx.check("mr_moe_combine_backward", st)
    return dys, dw


def _unchanged(ctx) -> None:
    if ctx.plan._version() != ctx.version:
        raise RuntimeError("the sorted tokens were modified by an inplace operation between "
                           "forward and backward")


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, plan):
        ctx.plan, ctx.version = plan, plan._version()
        return _dispatch(x, plan)

    @staticmethod
    @once_differentiable
    def backward(ctx, dxs):
        _unchanged(ctx)
        return moe_dispatch_backward(dxs, ctx.plan), None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ys, weights, plan, base):
        ctx.plan, ctx.version = plan, plan._version()
        ctx.save_for_backward(ys, weights)
        return _combine(ys, weights, plan, base)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        _unchanged(ctx)
        ys, weights = ctx.saved_tensors
        dys = dw = None
        if ctx.needs_input_grad[0] or ctx.needs_input_grad[1]:
            dys, dw = moe_combine_backward(dout, ys, weights, ctx.plan)
        return dys, dw, None, dout if ctx.needs_input_grad[3] else None


def _dual(*tensors) -> bool:
    """Whether one carries a forward-mode tangent (which the autograd functions refuse)."""
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def moe_dispatch(x: torch.Tensor, plan: SortedTokens) -> torch.Tensor:
    """``xs[r] = x[order[r] // top_k]`` [tokens * top_k, hidden]; rows without a pair are zero."""
    if (x.requires_grad and torch.is_grad_enabled()) or (
            forward_ad._current_level >= 0 and _dual(x)):
        return _Dispatch.apply(x, plan)
    return _dispatch(x, plan)


def moe_combine(ys: torch.Tensor, weights: torch.Tensor, plan: SortedTokens,
                base: torch.Tensor | None = None) -> torch.Tensor:
    """``out[t] = base[t] + sum_j weights[t, j] * ys[inverse[t, j]]``: fp32 sums in slot order,
    one rounding to the type of ``ys``. ``base``: rows to add (the shared expert's)."""
    if ((ys.requires_grad or weights.requires_grad or
         (base is not None and base.requires_grad)) and torch.is_grad_enabled()) or (
            forward_ad._current_level >= 0 and _dual(ys, weights, base)):
        return _Combine.apply(ys, weights, plan, base)
    return _combine(ys, weights, plan, base)
