"""Sorted tokens at the sizes that choose a kernel's form, on the GPU, against
the formulas in numpy and fp64."""
import ctypes as C

import numpy as np
import pytest
import torch

import minirun_moe as M
from minirun_moe import _lib as L

pytestmark = pytest.mark.gpu


def dev():
    return torch.device("cuda", 0)


def choice(T, k, E, seed, dropped):
    rng = np.random.default_rng(seed)
    ids = rng.integers(0, E, (T, k), dtype=np.int32)
    ids[rng.random((T, k)) < dropped] = -1
    return ids


def np_plan(ids, E):
    """order, inverse, offsets of a stable sort by expert."""
    key = np.where(ids.reshape(-1) >= 0, ids.reshape(-1), E)
    kept = np.argsort(key, kind="stable")[:(key < E).sum()]
    order = np.full(key.size, -1, np.int32)
    order[:len(kept)] = kept
    inverse = np.full(key.size, -1, np.int32)
    inverse[kept] = np.arange(len(kept), dtype=np.int32)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(key, minlength=E + 1)[:E])])
    return order, inverse.reshape(ids.shape), offsets


@pytest.mark.parametrize("E", [1, 5, 33, 100, 479, 999])
@pytest.mark.parametrize("T,k,dropped", [(4096, 1, 0.3), (4097, 1, 0.0), (1379, 3, 0.9),
                                         (4111, 7, 0.5), (65537, 1, 1.0)])
def test_sort_where_experts_end_inside_a_warp(T, k, E, dropped):
    """Expert counts that part a warp's lanes, pairs on both sides of one CTA's share."""
    ids = choice(T, k, E, T + E, dropped)
    p = M.moe_sort(torch.from_numpy(ids).to(dev()), E)
    order, inverse, offsets = np_plan(ids, E)
    np.testing.assert_array_equal(p.order.cpu().numpy(), order)
    np.testing.assert_array_equal(p.inverse.cpu().numpy(), inverse)
    np.testing.assert_array_equal(p.offsets.cpu().numpy(), offsets)
    assert M.Context.get(0).sync_check() == 0


def test_misaligned_pointers_are_refused():
    """Every int32 and fp32 pointer of the C entries two bytes off its alignment: refused before a
    launch."""
    T, k, E, H = 4, 2, 3, 64
    lib, ctx = L.load(), M.Context.get(0)
    ids = torch.zeros((T, k), dtype=torch.int32, device=dev())
    p = M.moe_sort(ids, E)
    x, ys = torch.zeros((T, H), device=dev()), torch.zeros((T * k, H), device=dev())
    w = torch.zeros((T, k), device=dev())
    mem = torch.zeros(2 * T * k + E + 1, dtype=torch.int32, device=dev())
    i, o = ids.data_ptr(), mem.data_ptr()
    n, f = o + 4 * T * k, o + 8 * T * k
    s = torch.cuda.current_stream().cuda_stream

    def refused(st):
        assert st == L.MR_ERR_INVALID_ARGUMENT
        assert b"aligned" in lib.mr_last_error(ctx.handle)

    for at in range(4):
        a = [q + 2 * (at == j) for j, q in enumerate((i, o, n, f))]
        refused(lib.mr_moe_sort(ctx.handle, a[0], T, k, E, a[1], a[2], a[3], s))
    for name in ("order", "inverse", "offsets"):
        c = L.mr_sorted.from_buffer_copy(p._c)
        setattr(c, name, getattr(c, name) + 2)
        ref = C.byref(c)
        X, Y, W, F = x.data_ptr(), ys.data_ptr(), w.data_ptr(), L.MR_DTYPE_F32
        refused(lib.mr_moe_dispatch(ctx.handle, X, F, H, H, ref, Y, s))
        refused(lib.mr_moe_dispatch_backward(ctx.handle, Y, F, H, H, ref, X, s))
        refused(lib.mr_moe_combine(ctx.handle, Y, F, H, H, W, None, ref, X, s))
        refused(lib.mr_moe_combine_backward(ctx.handle, X, H, Y, H, F, H, W, ref, Y, W, s))
        q = M.mxfp4_quantize(x)
        stack = M.mxfp4_quantize(torch.zeros((E, 32, H), device=dev()))
        refused(lib.mr_mxfp4_grouped_mm(ctx.handle, C.byref(q.desc()), C.byref(stack.desc()), ref,
                                        1, F, Y, s))
    ref = C.byref(p._c)
    refused(lib.mr_moe_combine(ctx.handle, Y, F, H, H, W + 2, None, ref, X, s))
    for a, b in ((2, 0), (0, 2)):
        refused(lib.mr_moe_combine_backward(ctx.handle, X, H, Y, H, F, H, W + a, ref, Y, W + b, s))


@pytest.mark.parametrize("bad", [2 ** 32 + 3, 2 ** 32, 2 ** 31, 2 ** 32 - 1, -2, -2 ** 31 - 1,
                                 -2 ** 32 - 1, -2 ** 63, 2 ** 63 - 1])
def test_int64_ids_out_of_range_are_reported_and_dropped(bad):
    ids = torch.tensor([[0, 3], [bad, 1], [-1, 3]], device=dev())
    p = M.moe_sort(ids, 4)
    assert p.inverse.tolist() == [[0, 2], [-1, 1], [-1, 3]]
    assert p.offsets.tolist() == [0, 1, 2, 2, 4] and p.order.tolist() == [0, 3, 1, 5, -1, -1]
    with pytest.raises(M.MoeError, match="expert id out of range"):
        M.Context.get(0).sync_check()
    M.moe_sort(torch.tensor([[0, -1]], device=dev()), 4)
    assert M.Context.get(0).sync_check() == 0


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_counts_of_experts_that_are_none(dtype):
    ids = torch.zeros((4, 2), dtype=dtype, device=dev())
    for experts in (2 ** 32 + 3, 2 ** 31, -2 ** 31 - 1):
        with pytest.raises(M.AffineBridgeError, match="32 bits"):
            M.moe_sort(ids, experts)
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    for experts in (0, -1, 1025, 2 ** 31 - 1):
        with pytest.raises(M.MoeError):
            M.moe_sort(ids, experts)
    assert torch.cuda.max_memory_allocated() - before < 1 << 20
    with pytest.raises(TypeError):
        M.moe_sort(ids, 3.0)


def test_a_values_flag_without_a_truth_value():
    x = torch.zeros((2, 64), device=dev())
    with pytest.raises(RuntimeError, match="ambiguous"):
        M.mxfp4_quantize(x, values=torch.zeros(2))


def test_without_the_short_way_the_results_are_the_same(monkeypatch):
    T, k, E, H, I = 40, 3, 6, 128, 64
    ids = torch.from_numpy(choice(T, k, E, 1, 0.2)).to(dev())
    x = torch.randn((T, H), generator=torch.Generator().manual_seed(2)).bfloat16().to(dev())
    w = torch.rand((T, k), generator=torch.Generator().manual_seed(3)).to(dev())
    stack = M.mxfp4_quantize(torch.randn((E, 2 * I, H), device=dev()))
    one = M.MXFP4Weights(stack.packed[0], stack.scales[0])

    def everything():
        p = M.moe_sort(ids, E)
        xs = M.moe_dispatch(x, p)
        q, v = M.mxfp4_quantize(x, values=True)
        mid = M.mxfp4_grouped_mm(q, stack, p, by_token=True)
        h = M.mxfp4_quantize_swiglu(mid)
        return (p.order, p.inverse, p.offsets, xs, M.moe_combine(xs, w, p),
                M.moe_dispatch_backward(xs, p), *M.moe_combine_backward(x, xs, w, p), q.packed,
                q.scales, v, mid, h.packed, h.scales, M.mxfp4_scaled_mm(q, one))

    first = everything()
    monkeypatch.setattr(L, "_torch_ext", L._NoShortWay())
    for a, b in zip(first, everything(), strict=True):
        assert torch.equal(a, b)


HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def within(got, ref, mag, n, dtype):
    """An fp32 sum of n products is within n * 2^-24 of their magnitudes' sum in any order; the
    result's rounding adds half an ulp (and half an f16 subnormal step)."""
    tol = (n + 2) * 2.0 ** -24 * mag + HALF_ULP[dtype] * (ref.abs() + mag * 2.0 ** -20)
    over = (got.double() - ref).abs() - tol - (2.0 ** -25 if dtype == torch.float16 else 0)
    assert bool((over <= 0).all()), float(over.max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,k,H", [
    (20011, 8, 96), (20011, 11, 96), (20011, 8, 131), (20011, 11, 131),  # eight slots a group
    (6007, 8, 96), (401, 8, 2048), (401, 7, 2050),                       # four
    (1501, 9, 2048), (801, 3, 520), (3001, 16, 260),                     # rows of several warps
])
def test_gradients_of_many_tokens(T, k, H, dtype):
    """Batches that fill the GPU take several slots in one group of threads."""
    ids = choice(T, k, 37, T + k, 0.1)
    p = M.moe_sort(torch.from_numpy(ids).to(dev()), 37)
    g = torch.Generator(device=dev()).manual_seed(H)
    ys, dout = (torch.randn((n, H), generator=g, device=dev()).to(dtype) for n in (T * k, T))
    w = torch.rand((T, k), generator=g, device=dev()) + 0.1
    inv = torch.from_numpy(np_plan(ids, 37)[1]).to(dev()).long()
    out, dx = M.moe_combine(ys, w, p), M.moe_dispatch_backward(ys, p)
    dys, dw = M.moe_combine_backward(dout, ys, w, p)
    ref, mag, rx, mx = (torch.zeros((T, H), dtype=torch.float64, device=dev()) for _ in range(4))
    for j in range(k):  # one slot of all tokens after another
        held = inv[:, j] >= 0
        r = inv[held, j]
        y, d, wj = ys[r].double(), dout[held].double(), w[held, j].double().unsqueeze(1)
        ref[held] += wj * y
        mag[held] += wj * y.abs()
        rx[held] += y
        mx[held] += y.abs()
        within(dys[r], wj * d, (wj * d).abs(), 1, dtype)
        within(dw[held, j], (d * y).sum(1), (d * y).abs().sum(1), H, torch.float32)
        assert bool((dw[~held, j] == 0).all())
    assert bool((dys[int(p.offsets[-1]):] == 0).all())
    within(out, ref, mag, k, dtype)
    within(dx, rx, mx, k, dtype)
    again = M.moe_combine_backward(dout, ys, w, p)
    assert torch.equal(dys, again[0]) and torch.equal(dw, again[1])
