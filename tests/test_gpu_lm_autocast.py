"""A training step captured inside a caller's autocast, which ends before the replays."""
import pytest
import torch

from paper_01_anti_decoy_pnfirtau_amd.wikilm import GraphedStep, WikiLM, WikiLMConfig, make_optimizer, train_step

pytestmark = pytest.mark.gpu


def test_step_captured_inside_the_caller_s_autocast(dev):
    cfg = WikiLMConfig(d_model=64, n_heads=4, n_layers=2, d_ff=128, max_seq=128, dropout=0.0)
    xs = torch.randint(0, 997, (6, 4, 128), generator=torch.Generator().manual_seed(0)).to(dev)

    def model():
        torch.manual_seed(0)
        m = WikiLM(997, cfg, "pn_fir_tau_flash").to(dev)
        return m, make_optimizer(m, cfg, capturable=True)

    m, opt = model()
    want = [float(train_step(m, opt, x, amp=True)) for x in xs]
    m, opt = model()
    x = xs[0].clone()
    with torch.autocast("cuda", torch.bfloat16):
        step = GraphedStep(m, opt, x, amp=True, warmup=2)
    for i in range(6):
        junk = [torch.full((n,), 7.0, device=dev, dtype=torch.bfloat16) for n in (997 * 64, 192 * 64, 128 * 64, 64 * 64)]
        del junk
        x.copy_(xs[i])
        got = float(step.replay())
        assert abs(got - want[i]) <= 1e-3 * abs(want[i]), (i, got, want[i])  # as captured steps outside of one
