"""What the language model's operators take, refuse and ignore at their seams with autograd and the model's settings."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from paper_01_anti_decoy_pnfirtau_amd import gated_ffn, linear_cross_entropy
from paper_01_anti_decoy_pnfirtau_amd.wikilm import WikiLM, WikiLMConfig, lm_loss
from tests.helpers import seeded

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [5, 100])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_checkpoint_counts_only_where_something_is_kept(dev, T, dtype):
    """A call that records no gradient keeps nothing: "e4m3" changes nothing there, fp32 operands included (a model that is
    trained under autocast may be evaluated in fp32)."""
    x, w_in, w_down = (seeded(s, 400 + i, dtype, dev) for i, s in enumerate(((T, 24), (32, 24), (24, 16))))
    assert torch.equal(gated_ffn(x, w_in, w_down, checkpoint="e4m3"), gated_ffn(x, w_in, w_down))
    with torch.no_grad():
        leaf = x.clone().requires_grad_()
        assert torch.equal(gated_ffn(leaf, w_in, w_down, checkpoint="e4m3"), gated_ffn(leaf, w_in, w_down))


def test_model_with_eight_bit_checkpoints_evaluates_in_fp32(dev):
    torch.manual_seed(0)
    m = WikiLM(100, WikiLMConfig(d_model=64, n_heads=4, n_layers=1, d_ff=96, max_seq=64, dropout=0.0, ffn="swiglu",
                                 ffn_checkpoint="e4m3", fused_loss=True), "pn_fir_tau_flash").to(dev)
    x = torch.randint(0, 100, (2, 64), generator=torch.Generator().manual_seed(1)).to(dev)
    with torch.no_grad():
        assert bool(lm_loss(m, x, amp=False).isfinite())
    with pytest.raises(ValueError, match="8-bit"):
        lm_loss(m, x, amp=False)
    assert bool(torch.cat([g.flatten() for g in torch.autograd.grad(lm_loss(m, x, amp=True), list(m.parameters()))]).isfinite().all())


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("leaf", [True, False])
def test_tangents_are_refused(dev, leaf, grad):
    """Forward mode: no tangent is dropped without a word, with and without a gradient recorded beside."""
    x, w_in, w_down, w = (seeded(s, 410 + i, torch.float32, dev) for i, s in enumerate(((4, 8), (12, 8), (8, 6), (10, 8))))
    target = torch.arange(4, device=dev)
    with fwd.dual_level(), torch.set_grad_enabled(grad):
        dual = fwd.make_dual(x.clone().requires_grad_(leaf), torch.ones_like(x))
        for call in (lambda: gated_ffn(dual, w_in, w_down), lambda: linear_cross_entropy(dual, w, target)):
            with pytest.raises((RuntimeError, ValueError)):
                call()
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: linear_cross_entropy(t, w, target), (x,), (x,))
