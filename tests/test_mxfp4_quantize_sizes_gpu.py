"""Quantisation to MXFP4 at the sizes where a thread takes several octets of
elements, on the GPU, against fp64: codes, exponents and values are equal."""
import pytest
import torch

import minirun_moe as M

pytestmark = pytest.mark.gpu

ROWS, WIDTH = 4801, 2080  # just past the size that fills the GPU, the last CTA nearly empty


def quantize_64(x):
    """(values, e8m0 exponents) of fp64 rows."""
    b = x.reshape(-1, 32)
    most = b.abs().amax(1)
    e = (torch.frexp(most)[1].long() - 3).clamp(-127, 127)
    e = torch.where(most == 0, -127, e).unsqueeze(1)
    two = ((e + 1023) << 52).view(torch.float64)  # 2^e
    u = (b / two).abs().clamp(max=6.0)
    step = torch.where(u < 2, 0.5, torch.where(u < 4, 1.0, 2.0)).double()
    v = torch.copysign(torch.round(u / step) * step * two, b)
    return v.reshape(x.shape), (e + 127).reshape(x.shape[0], -1)


def inputs(rows, width, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((rows, width), generator=g, device="cuda")
    return (x * torch.exp(torch.randn((rows, 1), generator=g, device="cuda"))).to(dtype)


def values_of(q):
    lut = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device="cuda")
    lut = torch.cat([lut, -lut])
    code = (q.packed.long().unsqueeze(-1) >> torch.arange(0, 32, 4, device="cuda")) & 15
    two = ((q.scales.long() + (1023 - 127)) << 52).view(torch.float64)
    return lut[code.flatten(-2)] * two.repeat_interleave(32, dim=-1)


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quantize(dtype, offset):
    x = inputs(ROWS, WIDTH + 3 * offset, dtype, 1)[:, offset:offset + WIDTH]
    q, values = M.mxfp4_quantize(x, values=True)
    v, e = quantize_64(x.double())
    assert torch.equal(q.scales.long(), e)
    assert torch.equal(values_of(q), v)
    assert torch.equal(values, v.float().to(dtype))


@pytest.mark.parametrize("limit", [0.0, 2.0])
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_swiglu(dtype, offset, limit):
    """h is within 2^-20: equal codes wherever that does not reach a rounding boundary."""
    x = inputs(ROWS, 2 * WIDTH + 3 * offset, dtype, 2)[:, offset:offset + 2 * WIDTH]
    gate, up = x.double().chunk(2, dim=1)
    if limit:
        gate, up = gate.clamp(max=limit), up.clamp(-limit, limit)
    h = gate / (1 + torch.exp(-gate)) * up
    q = M.mxfp4_quantize_swiglu(x, limit=limit)
    (lo, elo), (hi, ehi) = (quantize_64(h * f) for f in (1 - 2.0 ** -20, 1 + 2.0 ** -20))
    sure = (lo == hi) & (elo == ehi).repeat_interleave(32, dim=-1)
    assert float(sure.double().mean()) > 0.99
    got = values_of(q)
    assert torch.equal(got[sure], lo[sure])
    step = ((torch.maximum(elo, ehi) + 896) << 52).view(torch.float64)
    assert bool(((got - h).abs() <= 2.001 * step.repeat_interleave(32, dim=-1)).all())
