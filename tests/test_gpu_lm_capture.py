"""Captured steps of a model on a device that need not be the current one."""
import pytest
import torch

from paper_01_anti_decoy_pnfirtau_amd.wikilm import Decoder, GraphedStep, WikiLM, WikiLMConfig, make_optimizer

pytestmark = pytest.mark.gpu


def model(dev):
    torch.manual_seed(0)
    return WikiLM(97, WikiLMConfig(d_model=64, n_heads=2, n_layers=1, d_ff=96, max_seq=64, dropout=0.0)).to(dev)


def steps(dev):
    """A captured decoder's tokens and a captured training step's loss."""
    dec = Decoder(model(dev).eval(), 2, graph=True, temperature=0.0)
    dec.prefill(torch.arange(10, device=dev).view(2, 5))
    tokens = [dec.step(torch.zeros(2, device=dev)).tolist() for _ in range(4)]
    m, x = model(dev), torch.arange(64, device=dev).view(2, 32)
    return tokens, float(GraphedStep(m, make_optimizer(m, m.cfg, capturable=True), x, warmup=1).replay())


def test_the_model_s_device_is_current_in_a_capture(dev, monkeypatch):
    entered, graph, at = [], torch.cuda.graph, []

    class Device(torch.cuda.device):
        def __enter__(self):
            entered.append(self.idx)
            return super().__enter__()

        def __exit__(self, *args):
            entered.pop()
            return super().__exit__(*args)

    def spy(*args, **kwargs):
        at.append(list(entered))
        return graph(*args, **kwargs)

    monkeypatch.setattr(torch.cuda, "device", Device), monkeypatch.setattr(torch.cuda, "graph", spy)
    steps(dev)
    assert len(at) == 2 and all(dev.index in x for x in at)


@pytest.mark.skipif("torch.cuda.device_count() < 2", reason="one device")
def test_captures_on_another_device(dev):
    a, b = steps(dev), steps(torch.device("cuda:1"))
    assert a[0] == b[0] and abs(a[1] - b[1]) <= 1e-3 * abs(a[1])
