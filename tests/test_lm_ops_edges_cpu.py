"""The feed-forward block and the vocabulary cross entropy without a GPU: rows that are ignored."""
import pytest
import torch

import paper_01_anti_decoy_pnfirtau_amd as P


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_ignored_rows_reach_nothing_on_cpu(reduction):
    """As on the GPU: a row that is ignored may hold anything, and its loss and gradient are zero."""
    g = torch.Generator().manual_seed(0)
    x, w = torch.randn(2, 6, 8, generator=g), torch.randn(11, 8, generator=g)
    target = torch.tensor([[7, 3, 7, 10, 1, 7], [2, 7, 4, 4, 0, 7]])
    kept = target != 7
    x[~kept] = float("nan")
    x[0, 0], x[1, 5] = float("inf"), torch.finfo(torch.float32).min
    leaves, dense = ([t.clone().requires_grad_() for t in ts] for ts in ((x, w), (x[kept], w)))
    loss = P.linear_cross_entropy(*leaves, target, ignore_index=7, reduction=reduction)
    ref = P.linear_cross_entropy(*dense, target[kept], ignore_index=7, reduction=reduction)
    dx, dw = torch.autograd.grad(loss.sum(), leaves)
    rdx, rdw = torch.autograd.grad(ref.sum(), dense)
    if reduction == "none":
        assert not bool(loss[~kept].any())
        loss, ref = loss[kept], ref
    for a, b in ((loss, ref), (dx[kept], rdx), (dw, rdw)):
        assert torch.allclose(a, b, rtol=1e-6, atol=1e-6)
    assert not bool(dx[~kept].any())
