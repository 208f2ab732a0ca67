"""The 4-bit MoE layer's devices, without a GPU: what it refuses and where it launches."""
import contextlib
import types

import pytest
import torch

import minirun_moe as M
from minirun_moe import mxfp4_moe

E, H, I = 4, 64, 32


def matrix(out, width, experts=None, device="cpu", scales=None):
    lead = (experts, out) if experts else (out,)
    return M.MXFP4Weights(
        torch.zeros(lead + (width // 8,), dtype=torch.int32, device=device),
        torch.zeros(lead + (width // 32,), dtype=torch.uint8, device=scales or device))


def layer(router="cpu", gate_up="cpu", down="cpu", shared=None, **kw):
    return M.MXFP4MoELayer(torch.zeros((E, H), dtype=torch.bfloat16, device=router),
                           matrix(2 * I, H, E, gate_up, **kw), matrix(H, I, E, down),
                           M.RouterConfig.qwen(E, 2), shared)


def test_weights_on_two_devices_are_refused():
    layer()
    shared = (matrix(2 * I, H), matrix(H, I, device="meta"))
    for f in (lambda: layer(router="meta"), lambda: layer(gate_up="meta"),
              lambda: layer(down="meta"), lambda: layer(scales="meta"),
              lambda: layer(shared=shared)):
        with pytest.raises(M.AffineBridgeError, match="one device, got cpu, meta"):
            f()


def test_input_on_another_device_is_refused():
    with pytest.raises(M.AffineBridgeError, match="input is on meta, the layer on cpu"):
        layer()(torch.zeros((2, H), dtype=torch.bfloat16, device="meta"))


@pytest.mark.parametrize("current", [0, 1])
def test_every_step_runs_with_the_inputs_device_current(monkeypatch, current):
    now, seen = [current], []

    @contextlib.contextmanager
    def device(d):
        old, now[0] = now[0], d.index
        yield
        now[0] = old

    monkeypatch.setattr(torch.cuda, "current_device", lambda: now[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    sel = types.SimpleNamespace(ids=None, weights=None)
    for name in ("router_select", "moe_sort", "mxfp4_quantize", "mxfp4_grouped_mm",
                 "mxfp4_quantize_swiglu", "mxfp4_scaled_mm", "moe_combine"):
        monkeypatch.setattr(mxfp4_moe, name,
                            lambda *a, n=name, **k: (seen.append((n, now[0])), sel)[1])
    m = layer(shared=(matrix(2 * I, H), matrix(H, I)))
    m.device = torch.device("cuda", 1)
    m.forward(types.SimpleNamespace(dim=lambda: 2, shape=(2, H), dtype=torch.bfloat16,
                                    device=m.device, is_cuda=True))
    assert len(seen) == 10 and {d for _, d in seen} == {1}
    assert now[0] == current
