"""Tokens sorted by expert and back, on the GPU, against fp64 formulas.

Plans and copies are exact. Sums: an fp32 sum of n products is within n *
2^-24 of the sum of their magnitudes, times (1 + small), and rounding to the
result's type adds half an ulp (2^-8 for bf16, 2^-11 and half the subnormal
step, 2^-25, for f16, 2^-24 for fp32, relative).
"""
import ctypes as C

import numpy as np
import pytest
import torch

import minirun_moe as M
from minirun_moe import _lib as L

pytestmark = pytest.mark.gpu

HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def dev():
    return torch.device("cuda", 0)


def choice(T, k, E, seed, dropped=0.0, distinct=True):
    rng = np.random.default_rng(seed)
    if distinct and k <= E:
        ids = np.argsort(rng.random((T, E), dtype=np.float32), axis=1)[:, :k]
    else:
        ids = rng.integers(0, E, size=(T, k))
    ids = ids.astype(np.int32).reshape(T, k)
    ids[rng.random((T, k)) < dropped] = -1
    return ids


def np_plan(ids, E):
    flat = ids.reshape(-1)
    key = np.where((flat >= 0) & (flat < E), flat, E)
    kept = np.argsort(key, kind="stable")[:(key < E).sum()]
    order = np.full(flat.size, -1, np.int32)
    order[:len(kept)] = kept
    inverse = np.full(flat.size, -1, np.int32)
    inverse[kept] = np.arange(len(kept))
    counts = np.bincount(key, minlength=E + 1)[:E]
    return order, inverse.reshape(ids.shape), np.concatenate([[0], np.cumsum(counts)])


def rows(n, H, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn((n, H), generator=g).to(dtype).to(dev())


def f64(t):
    return t.double().cpu().numpy()


def within(got, ref, mag, n, dtype):
    """|got - ref| <= the bound above; mag: sum of the magnitudes."""
    err = np.abs(f64(got) - ref)
    tol = (n + 2) * 2.0 ** -24 * mag + HALF_ULP[dtype] * (np.abs(ref) + mag * 2.0 ** -20)
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25
    assert (err <= tol).all(), float((err - tol).max())


PLANS = [  # tokens, top_k, experts, dropped share
    (1, 1, 1, 0.0), (1, 8, 256, 0.0), (3, 2, 5, 0.5), (64, 8, 256, 0.0), (33, 4, 1024, 0.3),
    (513, 8, 60, 0.0), (512, 8, 61, 0.0), (4097, 3, 7, 0.2), (9001, 8, 256, 0.0),
    (700, 6, 1024, 1.0), (5, 32, 40, 0.1), (30011, 8, 1024, 0.1), (200003, 2, 3, 0.0),
]


@pytest.mark.parametrize("T,k,E,dropped", PLANS)
def test_sort_is_the_stable_order(T, k, E, dropped):
    ids = choice(T, k, E, T + k + E, dropped)
    p = M.moe_sort(torch.from_numpy(ids).to(dev()), E)
    order, inverse, offsets = np_plan(ids, E)
    np.testing.assert_array_equal(p.order.cpu().numpy(), order)
    np.testing.assert_array_equal(p.inverse.cpu().numpy(), inverse)
    np.testing.assert_array_equal(p.offsets.cpu().numpy(), offsets)
    assert M.Context.get(0).sync_check() == 0


def test_sort_one_expert_takes_everything():
    ids = np.full((3000, 4), 5, np.int32)
    p = M.moe_sort(torch.from_numpy(ids).to(dev()), 9)
    order, inverse, offsets = np_plan(ids, 9)
    np.testing.assert_array_equal(p.order.cpu().numpy(), order)
    np.testing.assert_array_equal(p.inverse.cpu().numpy(), inverse)
    np.testing.assert_array_equal(p.offsets.cpu().numpy(), offsets)


def test_sort_no_tokens():
    p = M.moe_sort(torch.zeros((0, 4), dtype=torch.int32, device=dev()), 300)
    assert p.offsets.cpu().tolist() == [0] * 301 and p.order.numel() == 0
    x = torch.zeros((0, 64), device=dev())
    assert M.moe_dispatch(x, p).shape == (0, 64)
    assert M.moe_combine(x, torch.zeros((0, 4), device=dev()), p).shape == (0, 64)


def test_sort_reports_ids_out_of_range_and_drops_them():
    ids = np.array([[0, 4], [7, 1], [-1, 3]], np.int32)
    p = M.moe_sort(torch.from_numpy(ids).to(dev()), 4)
    with pytest.raises(M.MoeError, match="expert id out of range"):
        M.Context.get(0).sync_check()
    ok = np.where((ids >= 0) & (ids < 4), ids, -1)
    np.testing.assert_array_equal(p.inverse.cpu().numpy(), np_plan(ok, 4)[1])


def test_sort_takes_int64_and_strided_ids():
    ids = choice(50, 8, 30, 3)
    wide = torch.from_numpy(ids.astype(np.int64)).to(dev())
    p = M.moe_sort(wide[:, ::2], 30)
    np.testing.assert_array_equal(p.order.cpu().numpy(), np_plan(ids[:, ::2], 30)[0])


WIDTHS = [1, 7, 64, 515, 1030, 2048, 7168]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H", WIDTHS)
def test_dispatch_copies_rows(dtype, H):
    T, k, E = 37, 3, 11
    ids = choice(T, k, E, H, 0.2)
    p = M.moe_sort(torch.from_numpy(ids).to(dev()), E)
    x = rows(T, H, dtype, H)
    xs = M.moe_dispatch(x, p)
    order = np_plan(ids, E)[0]
    ref = f64(x)[np.maximum(order, 0) // k] * (order >= 0)[:, None]
    np.testing.assert_array_equal(f64(xs), ref)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,T,k,E,dropped", [
    (1, 5, 2, 4, 0.0), (64, 1, 8, 16, 0.0), (515, 130, 3, 9, 0.4), (1030, 40, 6, 61, 0.2),
    (7168, 9, 8, 256, 0.0), (96, 1200, 12, 20, 0.1), (256, 3, 32, 40, 1.0),
])
def test_combine_and_gradients(dtype, H, T, k, E, dropped):
    ids = choice(T, k, E, H + T, dropped)
    p = M.moe_sort(torch.from_numpy(ids).to(dev()), E)
    inv = np_plan(ids, E)[1]
    held = inv >= 0
    ys, dout, base = rows(T * k, H, dtype, 1), rows(T, H, dtype, 2), rows(T, H, dtype, 3)
    w = torch.rand((T, k), generator=torch.Generator().manual_seed(4)).to(dev()) + 0.1
    yg = f64(ys)[np.maximum(inv, 0)] * held[..., None]
    wn, g = f64(w), f64(dout)

    ref = np.einsum("tk,tkh->th", wn, yg)
    mag = np.einsum("tk,tkh->th", wn, np.abs(yg))
    within(M.moe_combine(ys, w, p), ref, mag, k, dtype)
    within(M.moe_combine(ys, w, p, base=base), ref + f64(base), mag + np.abs(f64(base)), k + 1,
           dtype)
    within(M.moe_dispatch_backward(ys, p), yg.sum(1), np.abs(yg).sum(1), k, dtype)

    dys, dw = M.moe_combine_backward(dout, ys, w, p)
    ref = np.zeros((T * k, H))
    ref[inv[held]] = (wn[..., None] * g[:, None])[held]
    within(dys, ref, np.abs(ref), 1, dtype)
    # a thread's share of a row, then five shuffles and eight warps
    within(dw, np.einsum("th,tkh->tk", g, yg) * held,
           np.einsum("th,tkh->tk", np.abs(g), np.abs(yg)), H // 32 + 24, torch.float32)


def test_gradients_against_differences():
    """combine is linear in ys and in the weights, so a central difference of any step is its
    derivative; the dispatch is linear in x."""
    T, k, E, H = 21, 4, 6, 200
    ids = choice(T, k, E, 9, 0.2)
    p = M.moe_sort(torch.from_numpy(ids).to(dev()), E)
    ys, v, dout = (rows(T * k, H, torch.float32, 1), rows(T * k, H, torch.float32, 2),
                   rows(T, H, torch.float32, 3))
    w, u = (torch.rand((T, k), generator=torch.Generator().manual_seed(s)).to(dev()) + 0.1
            for s in (5, 6))
    dys, dw = M.moe_combine_backward(dout, ys, w, p)
    scale = T * k * H * 2.0 ** -22 * 8  # fp32 roundings of values of a few units
    by = (M.moe_combine(ys + v, w, p).double() - M.moe_combine(ys - v, w, p).double()) / 2
    held = (p.order >= 0).unsqueeze(1)
    assert abs(float((by * dout.double()).sum() - (dys.double() * v.double() * held).sum())) < scale
    by = (M.moe_combine(ys, w + u, p).double() - M.moe_combine(ys, w - u, p).double()) / 2
    assert abs(float((by * dout.double()).sum() - (dw.double() * u.double()).sum())) < scale
    x, d = rows(T, H, torch.float32, 7), rows(T, H, torch.float32, 8)
    by = (M.moe_dispatch(x + d, p).double() - M.moe_dispatch(x - d, p).double()) / 2
    dx = M.moe_dispatch_backward(ys, p)
    assert abs(float((by * ys.double()).sum() - (dx.double() * d.double()).sum())) < scale


def test_autograd_matches_the_functions():
    T, k, E, H = 30, 4, 8, 128
    p = M.moe_sort(torch.from_numpy(choice(T, k, E, 2, 0.1)).to(dev()), E)
    x = rows(T, H, torch.float32, 1).requires_grad_()
    w = (torch.rand((T, k), generator=torch.Generator().manual_seed(3)) + 0.1).to(dev())
    w.requires_grad_()
    base = rows(T, H, torch.float32, 4).requires_grad_()
    xs = M.moe_dispatch(x, p)
    out = M.moe_combine(xs, w, p, base=base)
    dout = rows(T, H, torch.float32, 5)
    out.backward(dout)
    dys, dw = M.moe_combine_backward(dout, xs.detach(), w.detach(), p)
    assert torch.equal(w.grad, dw) and torch.equal(base.grad, dout)
    assert torch.equal(x.grad, M.moe_dispatch_backward(dys, p))


def test_gradients_of_gradients_raise():
    p = M.moe_sort(torch.from_numpy(choice(6, 2, 4, 3)).to(dev()), 4)
    x = rows(6, 32, torch.float32, 1).requires_grad_()
    w = torch.full((6, 2), 0.5, device=dev(), requires_grad=True)
    (dx,) = torch.autograd.grad((M.moe_combine(M.moe_dispatch(x, p), w, p) ** 2).sum(), x,
                                create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


def test_strided_rows_match_contiguous_ones():
    """Rows that are slices of wider ones, at every alignment of the row."""
    T, k, E = 19, 2, 5
    p = M.moe_sort(torch.from_numpy(choice(T, k, E, 4)).to(dev()), E)
    w = torch.rand((T, k), device=dev()) + 0.1
    for dtype in TYPES:
        for off, H, wide in [(0, 64, 80), (1, 64, 81), (4, 100, 120), (2, 30, 50)]:
            x = rows(T, wide, dtype, 1)[:, off:off + H]
            y = rows(T * k, wide, dtype, 2)[:, off:off + H]
            assert torch.equal(M.moe_dispatch(x, p), M.moe_dispatch(x.contiguous(), p))
            assert torch.equal(M.moe_combine(y, w, p), M.moe_combine(y.contiguous(), w, p))
            a, b = M.moe_combine_backward(x, y, w, p)
            c, d = M.moe_combine_backward(x.contiguous(), y.contiguous(), w, p)
            assert torch.equal(a, c)
            np.testing.assert_allclose(b.cpu(), d.cpu(), rtol=0, atol=H * 2.0 ** -20)
    t = rows(64, T, torch.float32, 3).t()  # rows that are not contiguous: copied
    assert torch.equal(M.moe_dispatch(t, p), M.moe_dispatch(t.contiguous(), p))


def test_nan_and_inf_stay_where_they_are():
    """A dropped slot's weight and a neighbour's infinities touch nothing else."""
    T, k, E, H = 4, 2, 3, 64
    ids = np.array([[0, 1], [-1, 2], [1, 2], [-1, -1]], np.int32)
    p = M.moe_sort(torch.from_numpy(ids).to(dev()), E)
    ys = rows(T * k, H, torch.float32, 1)
    w = torch.ones((T, k), device=dev())
    w[1, 0] = float("nan")
    w[3] = float("inf")
    bad = int(p.inverse[2, 0])
    ys[bad, 5] = float("inf")
    out = M.moe_combine(ys, w, p)
    assert torch.isinf(out[2, 5])
    out[2, 5] = 0
    assert torch.isfinite(out).all() and (out[3] == 0).all()
    dys, dw = M.moe_combine_backward(rows(T, H, torch.float32, 2), ys, w, p)
    assert dw[1, 0] == 0 and (dw[3] == 0).all() and torch.isfinite(dys).all()


def test_combine_into_its_own_base():
    """The C entry allows base == out."""
    T, k, E, H = 9, 2, 4, 96
    p = M.moe_sort(torch.from_numpy(choice(T, k, E, 1)).to(dev()), E)
    ys, base = rows(T * k, H, torch.bfloat16, 1), rows(T, H, torch.bfloat16, 2)
    w = torch.rand((T, k), device=dev())
    ref = M.moe_combine(ys, w, p, base=base)
    ctx = M.Context.get(0)
    ctx.check("mr_moe_combine", L.load().mr_moe_combine(
        ctx.handle, ys.data_ptr(), L.MR_DTYPE_BF16, H, H, w.data_ptr(), base.data_ptr(),
        C.byref(p._c), base.data_ptr(), torch.cuda.current_stream().cuda_stream))
    assert torch.equal(base, ref)


def test_on_another_stream_and_in_a_graph():
    T, k, E, H = 64, 8, 256, 512
    ids = torch.from_numpy(choice(T, k, E, 8)).to(dev())
    x = rows(T, H, torch.bfloat16, 1)
    w = torch.rand((T, k), device=dev())
    ref = M.moe_combine(M.moe_dispatch(x, M.moe_sort(ids, E)), w, M.moe_sort(ids, E))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        p = M.moe_sort(ids, E)
        got = M.moe_combine(M.moe_dispatch(x, p), w, p)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, ref)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        p = M.moe_sort(ids, E)
        got = M.moe_combine(M.moe_dispatch(x, p), w, p)
    ids.copy_(torch.from_numpy(choice(T, k, E, 18)).to(dev()))
    g.replay()
    p = M.moe_sort(ids, E)
    assert torch.equal(got, M.moe_combine(M.moe_dispatch(x, p), w, p))


def test_rows_past_four_gigabytes():
    """Sorted rows whose byte offsets pass 32 bits."""
    T, k, E, H = 65, 4, 3, 9_000_000
    ids = choice(T, k, E, 5, distinct=False)
    p = M.moe_sort(torch.from_numpy(ids).to(dev()), E)
    x = torch.randint(-100, 100, (T, H), dtype=torch.int16, device=dev()).view(torch.bfloat16)
    xs = M.moe_dispatch(x, p)
    order = np_plan(ids, E)[0]
    for r in (0, 130, 255, 259):
        assert torch.equal(xs[r].view(torch.int16), x[order[r] // k].view(torch.int16))
    del xs, x
    torch.cuda.empty_cache()


def test_refusals():
    ids = torch.zeros((4, 2), dtype=torch.int32, device=dev())
    p = M.moe_sort(ids, 3)
    x = torch.zeros((4, 64), device=dev())
    ys = torch.zeros((8, 64), device=dev())
    w = torch.zeros((4, 2), device=dev())
    bad = [
        lambda: M.moe_sort(ids.float(), 3), lambda: M.moe_sort(ids[0], 3),
        lambda: M.moe_sort(ids.cpu(), 3),
        lambda: M.moe_dispatch(x[:3], p), lambda: M.moe_dispatch(x.double(), p),
        lambda: M.moe_dispatch(x.cpu(), p), lambda: M.moe_combine(x, w, p),
        lambda: M.moe_combine(ys, w.half(), p), lambda: M.moe_combine(ys, w[:, :1], p),
        lambda: M.moe_combine(ys, w, p, base=x.half()),
        lambda: M.moe_combine_backward(x.half(), ys, w, p),
        lambda: M.moe_combine_backward(x[:, :32], ys, w, p),
        lambda: M.SortedTokens(p.order[:4], p.inverse, p.offsets, 3),
        lambda: M.SortedTokens(p.order, p.inverse, p.offsets, 4),
        lambda: M.SortedTokens(p.order.long(), p.inverse, p.offsets, 3),
    ]
    for f in bad:
        with pytest.raises(M.AffineBridgeError):
            f()
    for experts in (0, -1, 1025):
        with pytest.raises(M.MoeError):
            M.moe_sort(ids, experts)
    with pytest.raises(M.MoeError, match="hidden"):
        M.moe_dispatch(torch.zeros((4, 0), device=dev()), p)
