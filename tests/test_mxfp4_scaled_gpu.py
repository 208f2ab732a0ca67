"""4 bits on both sides, on the GPU, against fp64 formulas.

Quantisation is exact: codes, exponents and values equal the formula's. In a
product every e2m1 product and its scales are exact; the sum runs over in/64
tensor-core steps, each within 2^-22 of the magnitudes it adds (fp32 with
truncated alignment), and rounding to bf16 adds half an ulp, 2^-8.
"""
import numpy as np
import pytest
import torch

import minirun_moe as M
from minirun_moe import _lib as L

pytestmark = pytest.mark.gpu

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def dev():
    return torch.device("cuda", 0)


def np_quantize(x):
    """(codes [rows, n], exponents [rows, n / 32]) of fp64 rows."""
    b = x.reshape(x.shape[0], -1, 32)
    most = np.abs(b).max(-1)
    ok = np.isfinite(b).all(-1)
    _, top = np.frexp(np.where(ok & (most > 0), most, 1.0))
    e = np.clip(top - 1 - 2 + 127, 0, 254)
    e = np.where(most > 0, e, 0)
    m = np.abs(np.where(ok[..., None], b, 0.0)) * 2.0 ** (127.0 - e)[..., None]
    m = np.minimum(m, 6.0)
    step = np.where(m < 2, 0.5, np.where(m < 4, 1.0, 2.0))
    v = np.rint(m / step) * step  # ties to even multiples: the even codes
    code = np.searchsorted(GRID, v)
    code = code + 8 * (np.signbit(b) & ok[..., None])
    return code.reshape(x.shape), np.where(ok, e, 255)


def np_values(code, e):
    v = GRID[code & 7] * np.where(code & 8, -1.0, 1.0)
    scale = np.where(e == 255, np.nan, 2.0 ** (e.astype(np.float64) - 127))
    return v * np.repeat(scale, 32, axis=-1)


def np_codes(w):
    """codes and exponents of device weights, rows flattened."""
    p = w.packed.cpu().numpy().view(np.uint32).reshape(-1, w.in_features // 8)
    code = (p[..., None] >> (4 * np.arange(8, dtype=np.uint32))) & 15
    return (code.reshape(p.shape[0], -1).astype(np.int64),
            w.scales.cpu().numpy().astype(np.int64).reshape(p.shape[0], -1))


def weights(out, inn, seed, experts=None, lo=124, hi=131):
    rng = np.random.default_rng(seed)
    lead = (experts, out) if experts else (out,)
    packed = rng.integers(0, 2 ** 32, lead + (inn // 8,), dtype=np.uint32).view(np.int32)
    scales = rng.integers(lo, hi, lead + (inn // 32,)).astype(np.uint8)
    return M.MXFP4Weights(torch.from_numpy(packed).to(dev()), torch.from_numpy(scales).to(dev()))


def dense(w):
    """fp64 [rows, in] of a matrix or [E, out, in] of a stack."""
    v = np_values(*np_codes(w))
    return v if w.experts is None else v.reshape(w.experts, w.out_features, w.in_features)


def check_mm(got, ref, mag, inn):
    g = got.double().cpu().numpy()
    np.testing.assert_array_equal(np.isnan(g), np.isnan(ref))
    ok = ~np.isnan(ref)
    tol = (inn / 64 + 2) * 2.0 ** -22 * mag
    if got.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * (np.abs(ref) + tol)
    err = np.abs(g - ref)
    assert (err <= tol)[ok].all(), float((err - tol)[ok].max())


# ------------------------------------------------------------- quantisation

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,n", [(1, 32), (3, 96), (64, 7168), (257, 224), (1000, 2048)])
def test_quantize_is_the_formula(dtype, rows, n):
    g = torch.Generator().manual_seed(rows + n)
    x = torch.randn((rows, n), generator=g) * torch.exp(2 * torch.randn((rows, 1), generator=g))
    x = x.to(dtype).to(dev())
    q, values = M.mxfp4_quantize(x, values=True)
    code, e = np_quantize(x.double().cpu().numpy())
    got, ge = np_codes(q)
    np.testing.assert_array_equal(ge, e)
    np.testing.assert_array_equal(got, code)
    want = torch.from_numpy(np_values(code, e)).to(dtype)
    assert torch.equal(values.cpu(), want)
    assert torch.equal(M.mxfp4_quantize(x).packed, q.packed)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quantize_every_tie_and_extreme(dtype):
    """Every midpoint of the grid at many exponents, the largest and smallest numbers, zeros."""
    mids = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 6.0, 0.0, -0.0, 0.26, 0.74, 1.3])
    info = torch.finfo(dtype)
    top = int(np.floor(np.log2(info.max)))
    low = int(np.log2(info.tiny)) - 4
    rows = []
    for k in range(low, top - 2):
        rows.append(np.concatenate([[4.0], mids, -mids, np.zeros(3)]) * 2.0 ** k)
    rows.append(np.zeros(32))
    rows.append(np.full(32, -0.0))
    rows.append(np.full(32, info.max))
    rows.append(np.linspace(-info.max, info.max, 32))
    rows.append(np.full(32, info.tiny))
    x = torch.from_numpy(np.stack(rows)).to(dtype).to(dev())
    q = M.mxfp4_quantize(x)
    code, e = np_quantize(x.double().cpu().numpy())
    got, ge = np_codes(q)
    np.testing.assert_array_equal(ge, e)
    np.testing.assert_array_equal(got, code)


def test_quantize_marks_blocks_without_a_number():
    x = torch.ones((3, 96), device=dev())
    x[0, 5] = float("nan")
    x[1, 40] = float("inf")
    x[2, 95] = float("-inf")
    q, v = M.mxfp4_quantize(x, values=True)
    s = q.scales.cpu().numpy()
    bad = np.array([[1, 0, 0], [0, 1, 0], [0, 0, 1]], bool)
    assert (s[bad] == 255).all() and (s[~bad] == 125).all()
    nan = torch.isnan(v).cpu().numpy()
    np.testing.assert_array_equal(nan, np.repeat(bad, 32, axis=1))
    assert (v[~torch.isnan(v)] == 1).all()
    np.testing.assert_array_equal(torch.isnan(M.mxfp4_dequantize(q)).cpu().numpy(), nan)


def test_quantize_strides_alignment_stacks():
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        x = torch.randn((9, 200), device=dev()).to(dtype)
        for off in (0, 1, 4, 8):
            v = x[:, off:off + 128]
            a, b = M.mxfp4_quantize(v), M.mxfp4_quantize(v.contiguous())
            assert torch.equal(a.packed, b.packed) and torch.equal(a.scales, b.scales)
        t = torch.randn((64, 9), device=dev()).to(dtype).t()
        a, b = M.mxfp4_quantize(t), M.mxfp4_quantize(t.contiguous())
        assert torch.equal(a.packed, b.packed)
    x = torch.randn((3, 10, 64), device=dev())
    a, b = M.mxfp4_quantize(x), M.mxfp4_quantize(x.reshape(30, 64))
    assert a.experts == 3 and a.out_features == 10
    assert torch.equal(a.packed.reshape(30, 8), b.packed)
    e = M.mxfp4_quantize(torch.zeros((0, 64), device=dev()))
    assert e.out_features == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,inter,limit", [(1, 32, 0.0), (77, 2048, 0.0), (5, 96, 1.0)])
def test_quantize_swiglu(dtype, rows, inter, limit):
    """h has a few fp32 roundings, 2^-20 relative: a block whose codes differ from the formula's
    holds a number that near to a rounding boundary, so its values are compared with h instead:
    at most half a step off, plus that; other blocks are equal."""
    x = torch.randn((rows, 2 * inter), generator=torch.Generator().manual_seed(inter)).to(dtype)
    x = (2 * x).to(dev())
    q = M.mxfp4_quantize_swiglu(x, limit=limit)
    g, u = x.double().cpu().numpy()[:, :inter], x.double().cpu().numpy()[:, inter:]
    if limit:
        g, u = np.minimum(g, limit), np.clip(u, -limit, limit)
    h = g / (1 + np.exp(-g)) * u
    near = np.stack([np.stack(np_quantize(h * f)[:1])[0] for f in (1 - 2.0 ** -20, 1 + 2.0 ** -20)])
    exps = np.stack([np_quantize(h * f)[1] for f in (1 - 2.0 ** -20, 1 + 2.0 ** -20)])
    sure = (near[0] == near[1]) & np.repeat(exps[0] == exps[1], 32, axis=1)
    code, e = np_codes(q)
    assert sure.mean() > 0.99
    np.testing.assert_array_equal(np_values(code, e)[sure], np_values(near[0], exps[0])[sure])
    step = 2.0 ** (np.repeat(np.maximum(*exps), 32, axis=1) - 127.0)  # widest gap is 2 of these
    assert (np.abs(np_values(code, e) - h) <= 2.001 * step).all()


def test_quantize_swiglu_strided_input():
    x = torch.randn((6, 300), device=dev(), dtype=torch.bfloat16)
    for off in (0, 3, 8):
        v = x[:, off:off + 256]
        a, b = M.mxfp4_quantize_swiglu(v), M.mxfp4_quantize_swiglu(v.contiguous())
        assert torch.equal(a.packed, b.packed) and torch.equal(a.scales, b.scales)


# ----------------------------------------------------------------- products

@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,out,inn", [
    (1, 1, 32), (1, 200, 256), (3, 128, 64), (16, 129, 288), (17, 500, 512), (77, 2040, 1024),
    (130, 64, 96), (225, 256, 2048), (1000, 384, 7168), (33, 7, 4000),
])
def test_scaled_mm(rows, out, inn, out_dtype):
    a, w = weights(rows, inn, rows + 1), weights(out, inn, out + 2)
    A, W = dense(a), dense(w)
    check_mm(M.mxfp4_scaled_mm(a, w, out_dtype=out_dtype), A @ W.T, np.abs(A) @ np.abs(W).T, inn)
    assert M.Context.get(0).sync_check() == 0


@pytest.mark.parametrize("rows,out,inn", [
    (1, 130, 2048), (5, 2048, 7168), (64, 300, 4096), (70, 256, 2080), (100, 1000, 4096),
    (33, 128, 8160),
])
def test_scaled_mm_few_tiles_split_along_the_rows(rows, out, inn):
    """Long rows and few tiles: several CTAs share one, and always add up alike."""
    a, w = weights(rows, inn, rows + 3), weights(out, inn, out + 4)
    A, W = dense(a), dense(w)
    for dt in (torch.bfloat16, torch.float32):
        y = M.mxfp4_scaled_mm(a, w, out_dtype=dt)
        check_mm(y, A @ W.T, np.abs(A) @ np.abs(W).T, inn)
        assert torch.equal(y, M.mxfp4_scaled_mm(a, w, out_dtype=dt))
    assert M.Context.get(0).sync_check() == 0


def grouped(T, k, E, out, inn, by_token, seed=0, dropped=0.0, ids=None, out_dtype=torch.bfloat16):
    rng = np.random.default_rng(seed)
    if ids is None:
        ids = np.stack([rng.permutation(E)[:k] for _ in range(T)]).astype(np.int32)
        ids[rng.random(ids.shape) < dropped] = -1
    plan = M.moe_sort(torch.from_numpy(ids).to(dev()), E)
    a = weights(T if by_token else T * k, inn, seed + 1)
    w = weights(out, inn, seed + 2, experts=E)
    got = M.mxfp4_grouped_mm(a, w, plan, by_token=by_token, out_dtype=out_dtype)
    A, W = dense(a), dense(w)
    order, off = plan.order.cpu().numpy(), plan.offsets.cpu().numpy()
    ref, mag = np.zeros((T * k, out)), np.zeros((T * k, out))
    for e in range(E):
        r = np.arange(off[e], off[e + 1])
        rows = A[order[r] // k] if by_token else A[r]
        ref[r], mag[r] = rows @ W[e].T, np.abs(rows) @ np.abs(W[e]).T
    check_mm(got, ref, mag, inn)
    assert M.Context.get(0).sync_check() == 0


@pytest.mark.parametrize("by_token", [False, True])
@pytest.mark.parametrize("T,k,E,out,inn,dropped", [
    (1, 8, 256, 128, 512, 0.0), (5, 2, 4, 200, 288, 0.0), (64, 8, 40, 136, 256, 0.0),
    (300, 4, 6, 256, 1024, 0.3), (40, 6, 1024, 64, 64, 0.0), (700, 2, 3, 130, 2048, 0.0),
    (9, 3, 5, 128, 96, 1.0), (2, 1, 3, 256, 4096, 0.0), (3, 2, 4, 100, 6144, 0.3),
])
def test_grouped_mm(T, k, E, out, inn, dropped, by_token):
    grouped(T, k, E, out, inn, by_token, seed=T, dropped=dropped)
    if T == 5:
        grouped(T, k, E, out, inn, by_token, seed=T + 1, dropped=dropped, out_dtype=torch.float32)


@pytest.mark.parametrize("by_token", [False, True])
@pytest.mark.parametrize("T", [10, 20, 43, 85, 150])
def test_grouped_mm_every_tile_width(T, by_token):
    """Mean rows of 5 to 75 an expert: every width of a tile, over drawn and dropped rows."""
    grouped(T, 4, 8, 328, 1056, by_token, seed=T, dropped=0.05)


@pytest.mark.parametrize("by_token", [False, True])
def test_grouped_mm_uneven_experts(by_token):
    """One expert with nearly all rows (several tiles), some with one, some with none."""
    ids = np.zeros((900, 1), np.int32)
    ids[::97] = 3
    ids[450] = 6
    grouped(900, 1, 8, 192, 512, by_token, ids=ids)


def test_nan_exponents_poison_their_rows_only():
    a, w = weights(20, 512, 1), weights(150, 512, 2)
    a.scales[7, 3] = 255
    w.scales[140, 15] = 255
    y = M.mxfp4_scaled_mm(a, w)
    nan = torch.zeros((20, 150), dtype=torch.bool)
    nan[7] = True
    nan[:, 140] = True
    assert torch.equal(torch.isnan(y).cpu(), nan)


def test_extreme_exponents():
    """Scales whose product is far outside either one's middle, and the smallest, 2^-127."""
    a, w = weights(9, 256, 1, lo=0, hi=2), weights(40, 256, 2, lo=250, hi=254)
    A, W = dense(a), dense(w)
    check_mm(M.mxfp4_scaled_mm(a, w, out_dtype=torch.float32), A @ W.T, np.abs(A) @ np.abs(W).T,
             256)


def test_offset_operands():
    """Experts taken out of a stack and rows out of a batch: bases that are not the tensor's."""
    w = weights(48, 96, 3, experts=5)
    a = weights(30, 96, 4)
    one = M.MXFP4Weights(w.packed[3], w.scales[3])
    A, W = dense(a), dense(w)[3]
    check_mm(M.mxfp4_scaled_mm(a, one), A @ W.T, np.abs(A) @ np.abs(W).T, 96)
    part = M.MXFP4Weights(a.packed[7:19], a.scales[7:19])
    check_mm(M.mxfp4_scaled_mm(part, one), A[7:19] @ W.T, np.abs(A[7:19]) @ np.abs(W).T, 96)


def test_results_do_not_depend_on_the_run():
    a, w = weights(70, 2048, 1), weights(300, 2048, 2, experts=6)
    ids = torch.from_numpy(np.random.default_rng(1).integers(0, 6, (70, 2)).astype(np.int32))
    plan = M.moe_sort(ids.to(dev()), 6)
    first = M.mxfp4_grouped_mm(a, w, plan, by_token=True, out_dtype=torch.float32)
    for _ in range(5):
        assert torch.equal(first, M.mxfp4_grouped_mm(a, w, plan, by_token=True,
                                                     out_dtype=torch.float32))


def test_product_in_a_graph_on_another_stream():
    a, w = weights(24, 512, 1), weights(256, 512, 2)
    ref = M.mxfp4_scaled_mm(a, w)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = M.mxfp4_scaled_mm(a, w)
    g.replay()
    assert torch.equal(got, ref)
    b = weights(24, 512, 9)
    a.packed.copy_(b.packed)
    a.scales.copy_(b.scales)
    g.replay()
    assert torch.equal(got, M.mxfp4_scaled_mm(b, w))


def test_experts_block_end_to_end():
    """Sort, quantise, grouped gate/up, SwiGLU, grouped down, combine against the same steps in
    fp64 on the same 4-bit operands."""
    T, k, E, H, I = 50, 3, 6, 256, 128
    rng = np.random.default_rng(3)
    ids = np.stack([rng.permutation(E)[:k] for _ in range(T)]).astype(np.int32)
    x = torch.from_numpy(rng.standard_normal((T, H)).astype(np.float32)).bfloat16().to(dev())
    wt = torch.from_numpy(rng.random((T, k)).astype(np.float32)).to(dev())
    gu, dn = weights(2 * I, H, 5, experts=E, lo=119, hi=122), weights(H, I, 6, experts=E, lo=119,
                                                                    hi=122)
    plan = M.moe_sort(torch.from_numpy(ids).to(dev()), E)
    xq = M.mxfp4_quantize(x)
    mid = M.mxfp4_grouped_mm(xq, gu, plan, by_token=True)
    h = M.mxfp4_quantize_swiglu(mid)
    ys = M.mxfp4_grouped_mm(h, dn, plan)
    out = M.moe_combine(ys, wt, plan)
    X, G, D, Hq = dense(xq), dense(gu), dense(dn), dense(h)
    ref = np.zeros((T, H))
    inv = plan.inverse.cpu().numpy()
    for t in range(T):
        for j in range(k):
            e = ids[t, j]
            np.testing.assert_allclose(mid[inv[t, j]].double().cpu().numpy(), G[e] @ X[t],
                                       rtol=2.0 ** -8, atol=1e-5)
            ref[t] += float(wt[t, j]) * (D[e] @ Hq[inv[t, j]])
    err = np.abs(out.double().cpu().numpy() - ref)
    assert (err <= 2.0 ** -7 * np.abs(ref).max()).all()


def test_refusals():
    a, w, stack = weights(4, 64, 1), weights(8, 64, 2), weights(8, 64, 3, experts=3)
    plan = M.moe_sort(torch.zeros((4, 1), dtype=torch.int32, device=dev()), 3)
    bad = [
        lambda: M.mxfp4_quantize(torch.zeros((2, 40), device=dev())),
        lambda: M.mxfp4_quantize(torch.zeros((2, 0), device=dev())),
        lambda: M.mxfp4_quantize(torch.zeros((2, 64))),
        lambda: M.mxfp4_quantize(torch.zeros((2, 64), device=dev(), dtype=torch.int32)),
        lambda: M.mxfp4_quantize_swiglu(torch.zeros((2, 96), device=dev())),
        lambda: M.mxfp4_scaled_mm(a, stack), lambda: M.mxfp4_scaled_mm(stack, w),
        lambda: M.mxfp4_scaled_mm(a, weights(8, 96, 2)),
        lambda: M.mxfp4_scaled_mm(a, w, out_dtype=torch.float16),
        lambda: M.mxfp4_grouped_mm(a, w, plan),
        lambda: M.mxfp4_grouped_mm(a, weights(8, 64, 3, experts=4), plan),
        lambda: M.mxfp4_grouped_mm(weights(5, 64, 1), stack, plan),
        lambda: M.mxfp4_grouped_mm(weights(5, 64, 1), stack, plan, by_token=True),
    ]
    for f in bad:
        with pytest.raises(M.MXFP4BridgeError):
            f()
    with pytest.raises(M.MoeError) as e:
        M.mxfp4_quantize_swiglu(torch.zeros((2, 128), device=dev()), limit=-1.0)
    assert e.value.status == L.MR_ERR_INVALID_ARGUMENT
    odd = torch.empty(4 * 8 + 1, dtype=torch.int32, device=dev())[1:].view(4, 8)
    with pytest.raises(M.MoeError, match="16-byte aligned"):
        M.mxfp4_scaled_mm(M.MXFP4Weights(odd, a.scales), w)


@pytest.mark.parametrize("T,shared,limit", [(1, False, 0.0), (37, True, 0.0), (300, True, 2.0)])
def test_layer_is_its_steps_in_64_bits(T, shared, limit):
    """MXFP4MoELayer against the same steps in fp64 on the same weights. The layer rounds the
    gate/up result to bf16 and the hidden values to 4 bits, so fp64 takes its hidden codes from
    the layer's own gate/up values; the rest is held to the bf16 rounding of ys, the shared rows
    and the sum, 3 * 2^-8 of the magnitudes added."""
    E, k, H, I = 8, 3, 256, 128
    g = torch.Generator().manual_seed(T)
    rnd = lambda *s: (torch.randn(s, generator=g) / s[-1] ** 0.5).to(dev())  # noqa: E731
    router_w = rnd(E, H).bfloat16()
    dense_w = (rnd(E, I, H), rnd(E, I, H), rnd(E, H, I))
    sh = (rnd(2 * I, H), rnd(2 * I, H), rnd(H, 2 * I)) if shared else None
    layer = M.MXFP4MoELayer.from_dense(router_w, *dense_w, M.RouterConfig.qwen(E, k), shared=sh,
                                       swiglu_limit=limit)
    x = torch.randn((T, H), generator=g).bfloat16().to(dev())
    out, sel = layer(x)

    def mlp(gu, dn, rows):  # one expert on 4-bit rows, its gate/up rounded as the kernel's
        mid = torch.from_numpy(rows @ gu.T).to(torch.bfloat16).double().numpy()
        a, u = mid[:, :mid.shape[1] // 2], mid[:, mid.shape[1] // 2:]
        if limit:
            a, u = np.minimum(a, limit), np.clip(u, -limit, limit)
        h = np_values(*np_quantize(a / (1 + np.exp(-a)) * u))
        return h @ dn.T, np.abs(h) @ np.abs(dn).T

    X = dense(M.mxfp4_quantize(x))
    G, D = dense(layer.gate_up), dense(layer.down)
    ids, wt = sel.ids.cpu().numpy(), sel.weights.double().cpu().numpy()
    ref, mag = np.zeros((T, H)), np.zeros((T, H))
    for t in range(T):
        for j in range(k):
            y, m = mlp(G[ids[t, j]], D[ids[t, j]], X[t:t + 1])
            ref[t] += wt[t, j] * y[0]
            mag[t] += wt[t, j] * m[0]
    if shared:
        y, m = mlp(dense(layer.shared[0]), dense(layer.shared[1]), X)
        ref, mag = ref + y, mag + m
    err = np.abs(out.double().cpu().numpy() - ref)
    # a gate/up sum next to a bf16 or 4-bit rounding boundary may fall the other way in fp64:
    # one code step of one hidden value then, at most 2 / 6 of its block's largest number
    within = err <= 3 * 2.0 ** -8 * mag
    assert within.mean() > 0.99, within.mean()
    assert np.linalg.norm(err) <= 2.0 ** -7 * np.linalg.norm(ref)


def test_layer_refusals():
    E, H, I = 4, 64, 32
    r = M.RouterConfig.qwen(E, 2)
    gu, dn = weights(2 * I, H, 1, experts=E), weights(H, I, 2, experts=E)
    rw = torch.zeros((E, H), dtype=torch.bfloat16, device=dev())
    layer = M.MXFP4MoELayer(rw, gu, dn, r)
    for f in (lambda: M.MXFP4MoELayer(rw, dn, gu, r),
              lambda: M.MXFP4MoELayer(rw, gu, weights(H, I, 2, experts=3), r),
              lambda: M.MXFP4MoELayer(rw, gu, dn, r, shared=(gu, dn)),
              lambda: M.MXFP4MoELayer(rw, gu, dn, r, swiglu_limit=-1.0),
              lambda: layer(torch.zeros((2, H), device=dev()))):
        with pytest.raises(M.AffineBridgeError):
            f()
