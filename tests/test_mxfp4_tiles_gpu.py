"""MXFP4 x MXFP4 products at the sizes of tiles, on the GPU, against fp64.

The bound is that of a sum of exact products over in/64 tensor-core steps, each
within 2^-22 of the magnitudes it adds; rounding to bf16 adds half an ulp, 2^-8.
"""
import numpy as np
import pytest
import torch

import minirun_moe as M

pytestmark = pytest.mark.gpu

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def dev():
    return torch.device("cuda", 0)


def matrix(rows, width, seed, experts=None):
    g = torch.Generator(device=dev()).manual_seed(seed)
    lead = (experts, rows) if experts else (rows,)
    packed = torch.randint(0, 2 ** 32, lead + (width // 8,), generator=g, device=dev())
    scales = torch.randint(120, 127, lead + (width // 32,), generator=g, device=dev())
    return M.MXFP4Weights((packed - 2 ** 31).to(torch.int32), scales.to(torch.uint8))


def values(w):
    """The numbers of a matrix or a stack, fp64."""
    lut = torch.tensor(GRID + tuple(-v for v in GRID), dtype=torch.float64, device=dev())
    word = w.packed.long().unsqueeze(-1) >> torch.arange(0, 32, 4, device=dev())
    scale = ((w.scales.long() + (1023 - 127)) << 52).view(torch.float64)
    return lut[(word & 15).flatten(-2)] * scale.repeat_interleave(32, dim=-1)


def check(got, ref, mag, width):
    tol = (width / 64 + 2) * 2.0 ** -22 * mag
    if got.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * (ref.abs() + tol)
    over = (got.double() - ref).abs() - tol
    assert bool((over <= 0).all()), float(over.max())
    assert M.Context.get(0).sync_check() == 0


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [33, 64, 100, 177])  # one CTA a tile, and two
@pytest.mark.parametrize("out,width", [(1, 512), (136, 512), (250, 544), (303, 1024), (33, 96)])
def test_rows_of_weights_that_end_inside_a_warp(rows, out, width, out_dtype):
    """Several groups of 16 result rows where some lanes of a warp have no weight row."""
    a, w = matrix(rows, width, rows), matrix(out, width, out)
    A, W = values(a), values(w)
    y = M.mxfp4_scaled_mm(a, w, out_dtype=out_dtype)
    check(y, A @ W.T, A.abs() @ W.abs().T, width)


def sorted_rows(counts, top_k, seed, dropped=0):
    """A plan whose experts have these numbers of pairs, in random order, `dropped` slots more."""
    ids = np.concatenate([np.repeat(np.arange(len(counts)), counts), np.full(dropped, -1)])
    ids = np.concatenate([ids, np.full(-len(ids) % top_k, -1)]).astype(np.int32)
    ids = np.random.default_rng(seed).permutation(ids).reshape(-1, top_k)
    return M.moe_sort(torch.from_numpy(ids).to(dev()), len(counts))


def check_grouped(counts, out, width, by_token, seed, out_dtype=torch.bfloat16, top_k=2,
                  dropped=0):
    p = sorted_rows(counts, top_k, seed, dropped)
    a = matrix(p.tokens if by_token else p.rows, width, seed + 1)
    w = matrix(out, width, seed + 2, experts=len(counts))
    got = M.mxfp4_grouped_mm(a, w, p, by_token=by_token, out_dtype=out_dtype)
    A = values(a)
    ref = torch.zeros((p.rows, out), dtype=torch.float64, device=dev())
    mag = torch.zeros_like(ref)
    off, order = p.offsets.tolist(), p.order.long()
    for e in range(len(counts)):
        r = slice(off[e], off[e + 1])
        x = A[order[r] // top_k] if by_token else A[r]
        W = values(M.MXFP4Weights(w.packed[e], w.scales[e]))
        ref[r], mag[r] = x @ W.T, x.abs() @ W.abs().T
    check(got, ref, mag, width)
    return a, w, p, got


@pytest.mark.parametrize("by_token", [False, True])
@pytest.mark.parametrize("counts,out,width", [
    ([3, 0, 1], 256, 4096),           # four CTAs a tile
    ([0, 0, 0], 256, 4096),           # and none of them with one
    ([150, 90, 0, 200], 600, 1024),   # two CTAs a tile
    ([0, 0, 0, 0], 600, 1024),
])
def test_clusters_end_together(counts, out, width, by_token):
    """Tiles shared by a cluster's CTAs, call after call, with rows that no expert takes: always
    the same results."""
    a, w, p, first = check_grouped(counts, out, width, by_token, 7, dropped=400 if out == 600
                                   else 5)
    for _ in range(20):
        assert torch.equal(first, M.mxfp4_grouped_mm(a, w, p, by_token=by_token))
    assert bool((first[sum(counts):] == 0).all())


def uneven(experts, mean, seed):
    """Rows of each expert, from none to twice the mean."""
    n = np.random.default_rng(seed).integers(0, 2 * mean + 1, experts)
    n[seed % experts] = 0
    return n.tolist()


# Every CTA or pair of 148 SMs takes three tiles at least, so that both accumulators, the rings and
# the exponents loaded ahead are used again, for tiles whose widths differ.
PIPELINES = [  # experts, mean rows, weight rows, widths with aligned exponents and without
    (128, 4, 648, (512, 1056)),    # tiles of 16 rows
    (64, 8, 1160, (2048, 2080)),   # 32
    (32, 18, 2568, (1024, 1056)),  # 64
    (24, 36, 2600, (1024, 544)),   # 128, by pairs of CTAs
    (8, 200, 4680, (512, 544)),    # 176
]


@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("by_token", [False, True])
@pytest.mark.parametrize("experts,mean,out,widths", PIPELINES)
def test_many_tiles_a_cta(experts, mean, out, widths, by_token, aligned):
    width = widths[0 if aligned else 1]
    counts = uneven(experts, mean, experts + mean)
    check_grouped(counts, out, width, by_token, experts, dropped=experts // 4,
                  out_dtype=torch.float32 if by_token == aligned else torch.bfloat16)


@pytest.mark.parametrize("rows,out,width", [(1500, 9001, 512), (1500, 9001, 544),
                                            (1061, 6200, 3104), (1061, 6200, 2560)])
def test_many_tiles_of_one_matrix(rows, out, width):
    a, w = matrix(rows, width, 1), matrix(out, width, 2)
    A, W = values(a), values(w)
    check(M.mxfp4_scaled_mm(a, w), A @ W.T, A.abs() @ W.abs().T, width)
