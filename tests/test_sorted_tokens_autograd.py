"""What autograd sees of moe_dispatch and moe_combine, with the kernels replaced by torch
operations on the CPU."""
import pytest
import torch
from torch.autograd import forward_ad

import minirun_moe as M
from minirun_moe import sorted_tokens as S

T, K, E, H = 4, 2, 3, 8


@pytest.fixture
def plan(monkeypatch):
    """A plan of rows in token order, and kernels that follow its inverse."""
    P = T * K
    mem = torch.cat([torch.arange(P), torch.arange(P), torch.tensor([0, 3, 5, P])]).int()

    def combine(ys, weights, p, base):
        rows = ys[p.inverse.long()] * weights.unsqueeze(-1)
        return rows.sum(1) + (0 if base is None else base)

    monkeypatch.setattr(S, "_dispatch", lambda x, p: x[p.order.long() // K].detach())
    monkeypatch.setattr(S, "_combine", lambda *a: combine(*a).detach())
    monkeypatch.setattr(S, "moe_dispatch_backward", lambda g, p: g[p.inverse.long()].sum(1))
    monkeypatch.setattr(S, "moe_combine_backward", lambda g, ys, w, p: (
        (w.unsqueeze(-1) * g.unsqueeze(1)).reshape(P, H),
        (g.unsqueeze(1) * ys[p.inverse.long()]).sum(-1)))
    return S.SortedTokens._of(mem, T, K, E)


def test_gradients_flow(plan):
    x = torch.randn(T, H, requires_grad=True)
    w = torch.rand(T, K, requires_grad=True)
    base = torch.randn(T, H, requires_grad=True)
    M.moe_combine(M.moe_dispatch(x, plan), w, plan, base=base).sum().backward()
    torch.testing.assert_close(x.grad, w.detach().sum(1, keepdim=True).expand(T, H))
    torch.testing.assert_close(w.grad, x.detach().sum(1, keepdim=True).expand(T, K))
    assert torch.equal(base.grad, torch.ones(T, H))


@pytest.mark.parametrize("grad_mode", [True, False])
def test_forward_mode_raises(plan, grad_mode):
    """Tangents are not built; they must not get lost either, whether or not a gradient is
    recorded."""
    x, ys, w, base = (torch.randn(s) for s in ((T, H), (T * K, H), (T, K), (T, H)))
    with torch.set_grad_enabled(grad_mode), forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        for f in (lambda: M.moe_dispatch(dual(x), plan),
                  lambda: M.moe_combine(dual(ys), w, plan),
                  lambda: M.moe_combine(ys, dual(w), plan),
                  lambda: M.moe_combine(ys, w, plan, base=dual(base))):
            with pytest.raises((RuntimeError, NotImplementedError)):
                f()
        # tensors without a tangent go as ever
        assert M.moe_combine(M.moe_dispatch(x, plan), w, plan, base=base).shape == (T, H)


@pytest.mark.parametrize("part", ["order", "inverse", "offsets"])
def test_a_plan_written_before_the_backward_pass_raises(plan, part):
    for f in (lambda x: M.moe_dispatch(x, plan),
              lambda x: M.moe_combine(x.repeat(K, 1), torch.ones(T, K), plan)):
        x = torch.randn(T, H, requires_grad=True)
        y = f(x)
        getattr(plan, part).zero_()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


def test_a_plan_of_the_callers_own_tensors(plan):
    own = S.SortedTokens.__new__(S.SortedTokens)
    own._mem, own._views = None, (plan.order.clone(), plan.inverse.clone(), plan.offsets.clone())
    own._fill(*(t.data_ptr() for t in own._views), T, K, E, own._views[0].device)
    x = torch.randn(T, H, requires_grad=True)
    M.moe_dispatch(x, own).sum().backward()
    assert torch.equal(x.grad, torch.full((T, H), float(K)))
    y = M.moe_dispatch(x, own)
    own._views[1].add_(0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_a_plan_made_in_inference_mode(plan):
    with torch.inference_mode():
        p = S.SortedTokens._of(plan._mem.clone(), T, K, E)
    x = torch.randn(T, H, requires_grad=True)
    M.moe_combine(M.moe_dispatch(x, p), torch.ones(T, K), p).sum().backward()
    assert torch.equal(x.grad, torch.full((T, H), float(K)))
