"""Training steps inside a caller's autocast, on CPU tensors: the casts of the weights follow the optimizer."""
import contextlib

import torch

from paper_01_anti_decoy_pnfirtau_amd.wikilm import WikiLM, WikiLMConfig, make_optimizer, train_step


def test_steps_inside_the_caller_s_autocast():
    cfg = WikiLMConfig(d_model=32, n_heads=2, n_layers=2, d_ff=48, max_seq=40, dropout=0.0, lr=1e-2)
    xs = torch.randint(0, 97, (4, 2, 40), generator=torch.Generator().manual_seed(0))
    losses = []
    for outer in (False, True):
        torch.manual_seed(0)
        m = WikiLM(97, cfg, "pn_fir_tau")
        opt = make_optimizer(m, cfg)
        with torch.autocast("cpu", torch.bfloat16) if outer else contextlib.nullcontext():
            losses.append(torch.stack([train_step(m, opt, x, amp=True) for x in xs]))
    assert torch.equal(*losses)
