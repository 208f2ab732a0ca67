"""An MoE layer whose experts multiply 4 bits by 4 bits.

The layer of ``MoELayer`` (router, routed experts, shared expert) with MXFP4
weights and MXFP4 activations: the router runs on the bf16 tokens; the
(token, slot) pairs are sorted by expert; every token is quantised once and
the gate/up product reads the tokens' rows in place; silu(gate) * up is
quantised as it is formed; the down product's rows go back to their tokens,
weighted, on top of the shared expert's.

  router_select -> moe_sort -> mxfp4_quantize -> mxfp4_grouped_mm (by token)
  -> mxfp4_quantize_swiglu -> mxfp4_grouped_mm -> moe_combine

Weights after the down product, as QwenMoEBlock.forward
(Sources/ModelAdapters/Model/QwenMoEModel.swift:340-351).
"""
from __future__ import annotations

import torch

from .bridge import AffineBridgeError, Selection
from .moe import RouterConfig, router_select
from .mxfp4 import MXFP4Weights
from .mxfp4_scaled import (mxfp4_grouped_mm, mxfp4_quantize, mxfp4_quantize_swiglu,
                           mxfp4_scaled_mm)
from .sorted_tokens import moe_combine, moe_sort


class MXFP4MoELayer:
    """``gate_up``: MXFP4 stack [E, 2 * inter, hidden], gate rows first; ``down``: [E, hidden,
    inter]; ``shared``: (gate_up [2 * shared_inter, hidden], down [hidden, shared_inter]) or
    None; ``router_w`` bf16 [E, hidden]. All on one GPU, which need not be the current one."""

    def __init__(self, router_w: torch.Tensor, gate_up: MXFP4Weights, down: MXFP4Weights,
                 router: RouterConfig,
                 shared: tuple[MXFP4Weights, MXFP4Weights] | None = None,
                 swiglu_limit: float = 0.0):
        E, hidden, inter = router.experts, gate_up.in_features, down.in_features
        if gate_up.experts != E or down.experts != E:
            raise AffineBridgeError(
                f"expert stacks must hold {E} experts, got {gate_up.experts} and {down.experts}")
        if gate_up.out_features != 2 * inter or down.out_features != hidden:
            raise AffineBridgeError(
                f"gate_up must be [{E}, 2 * inter, hidden] and down [{E}, hidden, inter], got "
                f"[{gate_up.out_features}, {hidden}] and [{down.out_features}, {inter}]")
        if shared is not None and (
                shared[0].experts is not None or shared[1].experts is not None or
                shared[0].in_features != hidden or shared[1].out_features != hidden or
                shared[0].out_features != 2 * shared[1].in_features):
            raise AffineBridgeError("the shared expert must be single matrices "
                                    "[2 * shared_inter, hidden] and [hidden, shared_inter]")
        if swiglu_limit < 0:
            raise AffineBridgeError("SwiGLU limit must be >= 0 (0: off)")
        mats = (gate_up, down, *(shared or ()))
        devices = {router_w.device, *(t.device for m in mats for t in (m.packed, m.scales))}
        if len(devices) > 1:
            raise AffineBridgeError("router and expert weights must be on one device, got "
                                    + ", ".join(sorted(map(str, devices))))
        self.device = router_w.device
        self.router_w = router_w.contiguous()
        self.gate_up, self.down, self.router, self.shared = gate_up, down, router, shared
        self.swiglu_limit = float(swiglu_limit)
        self.hidden, self.inter = hidden, inter

    @staticmethod
    def from_dense(router_w: torch.Tensor, gate: torch.Tensor, up: torch.Tensor,
                   down: torch.Tensor, router: RouterConfig,
                   shared: tuple[torch.Tensor, torch.Tensor, torch.Tensor] | None = None,
                   swiglu_limit: float = 0.0) -> "MXFP4MoELayer":
        """Quantises bf16 / f16 / fp32 stacks gate, up [E, inter, hidden] and down [E, hidden,
        inter] (and the shared expert's gate, up, down matrices) on their GPU."""
        sh = None
        if shared is not None:
            sh = (mxfp4_quantize(torch.cat(shared[:2])), mxfp4_quantize(shared[2]))
        return MXFP4MoELayer(router_w, mxfp4_quantize(torch.cat((gate, up), dim=1)),
                             mxfp4_quantize(down), router, sh, swiglu_limit)

    def forward(self, x: torch.Tensor) -> tuple[torch.Tensor, Selection]:
        """bf16 [tokens, hidden] -> bf16 [tokens, hidden] and the router's selection."""
        if x.dim() != 2 or x.shape[1] != self.hidden or x.dtype != torch.bfloat16:
            raise AffineBridgeError(
                f"input must be a [tokens, {self.hidden}] bfloat16 matrix, got {list(x.shape)} "
                f"{x.dtype}")
        if x.device != self.device:
            raise AffineBridgeError(f"input is on {x.device}, the layer on {self.device}")
        if x.is_cuda and x.device.index != torch.cuda.current_device():
            # the router launches on the current device and its stream, the rest on x's
            with torch.cuda.device(x.device):
                return self._forward(x)
        return self._forward(x)

    def _forward(self, x: torch.Tensor) -> tuple[torch.Tensor, Selection]:
        sel = router_select(x, self.router_w, self.router)
        plan = moe_sort(sel.ids, self.router.experts)
        xq = mxfp4_quantize(x)
        mid = mxfp4_grouped_mm(xq, self.gate_up, plan, by_token=True)
        ys = mxfp4_grouped_mm(mxfp4_quantize_swiglu(mid, self.swiglu_limit), self.down, plan)
        base = None
        if self.shared is not None:
            h = mxfp4_quantize_swiglu(mxfp4_scaled_mm(xq, self.shared[0]), self.swiglu_limit)
            base = mxfp4_scaled_mm(h, self.shared[1])
        return moe_combine(ys, sel.weights, plan, base=base), sel

    __call__ = forward
