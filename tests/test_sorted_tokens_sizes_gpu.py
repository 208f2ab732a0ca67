"""Sorted tokens at the sizes that choose a kernel's form, on the GPU, against
the formulas in numpy and fp64."""
import numpy as np
import pytest
import torch

import minirun_moe as M

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
