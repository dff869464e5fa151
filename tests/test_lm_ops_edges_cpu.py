"""The feed-forward block and the vocabulary cross entropy without a GPU: rows that are ignored, what is kept, the workspaces'
sizes, and what the C ABI says of strides."""
import pytest
import torch

import paper_01_anti_decoy_pnfirtau_amd as P
from paper_01_anti_decoy_pnfirtau_amd import _lib


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


def test_cpu_tensors_take_flat_targets():
    """The rows of [B, N, D] against B N targets in a row, as F.cross_entropy takes flattened logits."""
    g = torch.Generator().manual_seed(4)
    x, w, target = torch.randn(2, 5, 8, generator=g), torch.randn(11, 8, generator=g), torch.arange(10)
    target[3] = -100
    assert torch.equal(P.linear_cross_entropy(x, w, target), P.linear_cross_entropy(x, w, target.view(2, 5)))
    assert P.linear_cross_entropy(x, w, target, reduction="none").shape == (10,)
    assert float(P.linear_cross_entropy(x[:0], w, target[:0].view(0, 5), reduction="sum")) == 0.0


@pytest.mark.parametrize("T,D,V,dtype", [(65536, 256, 65536, "bf16"), (16384, 256, 33278, "bf16"), (8192, 2048, 65536, "bf16"),
                                         (65536, 256, 65536, "f32"), (16384, 512, 40001, "f32")])
def test_cross_entropy_backward_workspace_is_a_piece_and_little_else(T, D, V, dtype):
    """A piece of d (256 MB, or 2048 tokens), the kept rows, fp32 sums of the two gradients, of two splits at most at these
    sizes, and a few words for each row: far from all of d.  A loss per row has the rows times their factors beside."""
    es, code = (2, _lib.PNFX_BF16) if dtype == "bf16" else (4, _lib.PNFX_F32)
    piece = max(256 << 20, 2048 * T * es)
    copies = D % 8 != 0
    mean, per_row = (_lib.lib().pnfx_xent_bwd_workspace_size(T, D, V, _lib.PNFX_REDUCE[r], copies, code) for r in ("mean", "none"))
    tokens = piece // (T * es)
    assert mean <= piece + T * D * es + 2 * T * D * 4 + 2 * tokens * D * 4 + 40 * T + 65536
    assert mean < T * V * es / 2
    assert per_row == mean + T * D * es
    assert _lib.lib().pnfx_xent_bwd_workspace_size(T, D, V, _lib.PNFX_REDUCE["sum"], copies, code) == mean


def test_cpu_tensors_keep_what_torch_keeps():
    """The CPU composition takes both checkpoint settings, which are the GPU kernel's, and gives the same gradients."""
    g = torch.Generator().manual_seed(3)
    for dtype in (torch.float32, torch.bfloat16):
        leaves = [torch.randn(s, generator=g).to(dtype).requires_grad_() for s in ((5, 8), (12, 8), (7, 6))]
        grads = [torch.autograd.grad(P.gated_ffn(*leaves, checkpoint=keep).sum(), leaves) for keep in ("full", "e4m3")]
        assert all(torch.equal(a, b) for a, b in zip(*grads))


def test_c_abi_names_bad_row_strides():
    import ctypes

    p, big, lib = ctypes.c_void_p(256), 1 << 40, _lib.lib()
    assert lib.pnfx_ffn_fwd(p, 15, p, 16, p, 8, p, p, p, 4, 16, 8, 16, 0, 1, 1, p, big, None) == -1
    assert b"row strides 15, 16, 8" in lib.pnfx_last_error()
    assert lib.pnfx_ffn_bwd(p, 15, p, 16, p, 16, p, 8, p, p, p, p, p, 4, 16, 8, 16, 0, 1, 1, p, big, None) == -1
    assert b"row strides 15, 16, 16, 8" in lib.pnfx_last_error()
    assert lib.pnfx_xent_fwd(p, 8, p, 16, p, -100, p, p, p, 4, 16, 20, 2, 1, p, big, None) == -1
    assert b"row strides 8, 16" in lib.pnfx_last_error()
