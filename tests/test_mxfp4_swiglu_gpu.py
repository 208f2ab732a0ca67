"""silu(gate) * up in MXFP4 over the whole range of gates, on the GPU, against fp64.

CUDA's expf is within 2 ulp (2^-22 relative), every other step of fp32 within
2^-24: in gate / (1 + exp(-gate)) * up that is 2^-22 + 3 * 2^-24, and where far
negative gates take exp(gate / 2) twice, 2 * 2^-22 + 3 * 2^-24. Both are below
2^-20, so codes are equal unless h is that near to a rounding boundary.
"""
import numpy as np
import pytest
import torch

import minirun_moe as M

pytestmark = pytest.mark.gpu

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def np_quantize(x):
    """Values of fp64 rows in MXFP4 and their blocks' exponents."""
    b = x.reshape(x.shape[0], -1, 32)
    most = np.abs(b).max(-1)
    _, top = np.frexp(most)
    e = np.where(most > 0, np.clip(top - 3, -127, 127), -127)[..., None]
    u = np.minimum(np.abs(np.ldexp(b, -e)), 6.0)
    step = np.where(u < 2, 0.5, np.where(u < 4, 1.0, 2.0))
    v = np.ldexp(np.sign(b) * np.rint(u / step) * step, e)
    return v.reshape(x.shape), e[..., 0]


def np_values(q):
    p = q.packed.cpu().numpy().view(np.uint32)
    code = ((p[..., None] >> (4 * np.arange(8, dtype=np.uint32))) & 15).reshape(p.shape[0], -1)
    e = q.scales.cpu().numpy().astype(np.int64) - 127
    v = GRID[code & 7] * np.where(code & 8, -1.0, 1.0)
    return np.ldexp(v, np.repeat(e, 32, axis=1)), e


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("scale", [1.0, 2.0 ** 60, 2.0 ** 120])
def test_every_gate_has_its_value(dtype, scale):
    """Blocks of gates half a unit wide, from -170 to 40: each with codes of its own exponent, down
    to the smallest that e8m0 has."""
    rng = np.random.default_rng(int(np.log2(scale)))
    mid = np.arange(-170, 40, 0.5)
    gate = mid[:, None] + rng.uniform(-0.25, 0.25, (len(mid), 64))
    up = rng.standard_normal((len(mid), 64)) * scale / np.maximum(1, np.abs(mid))[:, None]
    x = torch.from_numpy(np.concatenate([gate, up], axis=1)).to(dtype).cuda()
    g, u = x.double().cpu().numpy()[:, :64], x.double().cpu().numpy()[:, 64:]
    with np.errstate(over="ignore"):
        h = g / (1 + np.exp(-g)) * u
    got, e = np_values(M.mxfp4_quantize_swiglu(x))
    (lo, elo), (hi, ehi) = (np_quantize(h * f) for f in (1 - 2.0 ** -20, 1 + 2.0 ** -20))
    sure = (lo == hi) & np.repeat(elo == ehi, 32, axis=1)
    assert sure.mean() > 0.99
    np.testing.assert_array_equal(got[sure], lo[sure])
    step = np.ldexp(1.0, np.repeat(np.maximum(elo, ehi), 32, axis=1))
    assert (np.abs(got - h) <= 2.001 * step).all()


def test_gates_without_a_number():
    """-inf * 0 and NaN mark their block; +inf with any up but 0 as well."""
    x = torch.ones((4, 128), device="cuda")
    for r, v in enumerate((float("-inf"), float("inf"), float("nan"), -1e30)):
        x[r, 40] = v
    q = M.mxfp4_quantize_swiglu(x)
    assert q.scales.cpu().tolist() == [[124, 255]] * 3 + [[124, 124]]
