"""Layers and the language model over the 8-bit cache on the GPU: a run of its operators as they are used together."""
import contextlib

import pytest
import torch

from paper_01_anti_decoy_pnfirtau_amd import PnFirConfig, PnFirTauFlashMHA
from paper_01_anti_decoy_pnfirtau_amd.wikilm import Decoder, WikiLM, WikiLMConfig, generate

pytestmark = pytest.mark.gpu
WARM = 30.0  # of a new model, whose tied embeddings give the last token a logit of about d_model: draws that vary


def model(dev, **kw):
    torch.manual_seed(0)
    cfg = WikiLMConfig(d_model=128, n_heads=2, n_layers=3, d_ff=256, max_seq=128, dropout=0.0, **kw)
    return WikiLM(997, cfg, "pn_fir_tau_flash").eval().to(dev)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_layer_over_the_cache_is_the_dense_layer_up_to_8_bits(dev, dtype):
    torch.manual_seed(1)
    layer = PnFirTauFlashMHA(PnFirConfig(d_model=128, n_heads=2)).eval().to(dev, dtype)
    x = torch.randn(2, 200, 128, device=dev, dtype=dtype)
    with torch.no_grad():
        want = layer(x).float()
        cache = layer.new_cache(2, 200, page=32)
        got = torch.cat([layer.forward_cached(x[:, a:b], cache, a) for a, b in ((0, 117), (117, 118), (118, 200))], 1)
    assert (got.float() - want).norm() < 0.15 * want.norm()


@pytest.mark.parametrize("amp", [False, True])
def test_generate_same_as_the_cpu_one_and_captured(dev, amp):
    m = model(dev)
    g = torch.Generator().manual_seed(2)
    prompt = torch.randint(0, 997, (3, 20), generator=g)
    lengths, u = torch.tensor([20, 7, 1]), torch.rand(3, 30, generator=g)
    run = lambda **kw: generate(m, prompt.to(dev), 30, lengths.to(dev), u.to(dev), amp=amp, temperature=0.8,  # noqa: E731
                                top_k=100, top_p=0.95, **kw)
    eager = run()
    assert torch.equal(eager, run(graph=True))
    assert torch.equal(eager, run())
    assert 0 <= int(eager.min()) and int(eager.max()) < 997
    if not amp:
        with torch.no_grad():  # the logits of the prompts' last rows, on the GPU and the CPU
            on = m.head(m.hidden_cached(prompt.to(dev), m.new_caches(3), 0)).cpu()
            cpu = m.cpu()
            off = cpu.head(cpu.hidden_cached(prompt, cpu.new_caches(3), 0))
        assert (on - off).abs().max() < 1e-2 * off.abs().max()  # fp32 sums move some 8-bit roundings


def test_decoders_side_by_side(dev):
    """Two captured decoders, their replays and eager steps mixed, on two streams, and prompts taken anew."""
    m = model(dev)
    g = torch.Generator().manual_seed(4)
    prompts = [torch.randint(0, 997, (2, 15), generator=g).to(dev) for _ in range(2)]
    u = torch.rand(2, 24, 2, generator=g).to(dev)
    want = []
    for i in range(2):
        dec = Decoder(m, 2, temperature=0.9)
        dec.prefill(prompts[i])
        want.append(torch.stack([dec.step(u[i, t]).clone() for t in range(24)]))
    decs = [Decoder(m, 2, graph=True, temperature=0.9) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(2):
        got = [[], []]
        for i in range(2):
            decs[i].prefill(prompts[i])
        torch.cuda.synchronize()
        for t in range(24):
            for i in range(2):
                with torch.cuda.stream(streams[i]):
                    got[i].append(decs[i].step(u[i, t]).clone())
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(torch.stack(got[i]), want[i])


def test_captured_inside_the_caller_s_autocast(dev):
    """The captured step goes on after that context has ended, its memory has other contents and weights have changed."""
    m = model(dev)
    g = torch.Generator().manual_seed(5)
    prompt, u = torch.randint(0, 997, (2, 15), generator=g).to(dev), torch.rand(24, 2, generator=g).to(dev)

    def run(graph, outer):
        with torch.no_grad():
            m.blocks[1].attn.out.weight.copy_(weight)
        dec = Decoder(m, 2, amp=True, graph=graph, temperature=WARM)
        around = lambda: torch.autocast("cuda", torch.bfloat16) if outer else contextlib.nullcontext()  # noqa: E731
        with around():
            dec.prefill(prompt)
            got = [(dec.step(u[t]).clone(), dec.rows.clone()) for t in range(3)]
        for t in range(3, 24):
            junk = [torch.full((n,), 7.0, device=dev, dtype=torch.bfloat16) for n in (997 * 128, 384 * 128, 128 * 128, 256 * 128)]
            del junk
            if t == 9:
                with torch.no_grad():
                    m.blocks[1].attn.out.weight.mul_(-2)
            got.append((dec.step(u[t]).clone(), dec.rows.clone()))
        with around():  # a replay inside another one
            got.append((dec.step(u[0]).clone(), dec.rows.clone()))
        return [torch.stack(x) for x in zip(*got)]

    weight = m.blocks[1].attn.out.weight.detach().clone()
    want = run(False, False)
    assert len(want[0].unique()) > 24  # draws of many tokens
    for kind in ((False, True), (True, True), (True, False)):
        assert all(torch.equal(a, b) for a, b in zip(run(*kind), want))


def test_sequences_that_begin_below_zero(dev):
    """They get NaN, as from the cache, and their neighbours what they get alone."""
    m, idx = model(dev), torch.randint(0, 997, (2, 3), generator=torch.Generator().manual_seed(6)).to(dev)
    with torch.no_grad():
        got = m.hidden_cached(idx, m.new_caches(2), torch.tensor([-7, 0], dtype=torch.int32, device=dev))
        want = m.hidden_cached(idx, m.new_caches(2), 0)
    assert got[0].isnan().all() and torch.equal(got[1], want[1])


def test_positions_that_the_model_does_not_have(dev):
    m = WikiLM(97, WikiLMConfig(d_model=64, n_heads=2, n_layers=2, d_ff=96, max_seq=40, dropout=0.0)).eval().to(dev)
    idx, start = torch.randint(0, 97, (2, 3), device=dev), torch.tensor([39, 4], dtype=torch.int32, device=dev)
    with torch.no_grad():
        got = m.hidden_cached(idx, m.new_caches(2), start)
        with pytest.raises(ValueError, match="hidden_cached"):
            m.hidden_cached(idx, m.new_caches(2), 38)
    assert got[0, 0].isfinite().all() and got[0, 1:].isnan().all() and got[1].isfinite().all()


@pytest.mark.parametrize("graph", [False, True])
def test_lengths_outside_their_prompts(dev, graph):
    """Known on the host: refused; on the device: -1 for those sequences, and their neighbours go on."""
    m, g = model(dev), torch.Generator().manual_seed(8)
    prompt, u = torch.randint(0, 997, (4, 9), generator=g).to(dev), torch.rand(6, 4, generator=g).to(dev)
    dec = Decoder(m, 4, graph=graph, temperature=WARM)
    with pytest.raises(ValueError, match="lengths"):
        dec.prefill(prompt, torch.tensor([9, 0, 10, 2]))

    def run(lengths):
        dec.prefill(prompt, lengths)
        return torch.stack([dec.step(x).clone() for x in u])

    got, want = run(torch.tensor([9, 0, 10, 2], device=dev)), run(torch.tensor([9, 1, 9, 2]))
    assert (got[:, 1:3] == -1).all() and torch.equal(got[:, [0, 3]], want[:, [0, 3]]) and want.min() >= 0


@pytest.mark.parametrize("kinds", [(torch.float32, torch.int32), (torch.float64, torch.int64)])
def test_settings_that_change_between_captured_steps(dev, kinds):
    m, g = model(dev), torch.Generator().manual_seed(9)
    prompt, u = torch.randint(0, 997, (3, 9), generator=g).to(dev), torch.rand(12, 3, generator=g).to(dev)

    def run(graph):
        temperature, top_p = (torch.full((3,), x, dtype=kinds[0], device=dev) for x in (WARM, 0.9))
        top_k = torch.full((3,), 50, dtype=kinds[1], device=dev)
        dec = Decoder(m, 3, graph=graph, temperature=temperature, top_p=top_p, top_k=top_k)
        dec.prefill(prompt)
        out = []
        for t, x in enumerate(u):
            temperature.fill_(WARM + 2 * t), top_k.fill_(50 + 400 * (t % 3)), top_p.fill_(1.0 if t % 2 else 0.8)
            out.append(dec.step(x).clone())
        return torch.stack(out)

    want = run(False)
    assert torch.equal(run(True), want) and len(want.unique()) > 20


def test_in_inference_mode(dev):
    m, prompt = model(dev), torch.randint(0, 997, (2, 9), generator=torch.Generator().manual_seed(1)).to(dev)
    u = torch.rand(2, 6, generator=torch.Generator().manual_seed(2)).to(dev)
    want = generate(m, prompt, 6, u=u, temperature=WARM)
    with torch.inference_mode():
        for graph in (False, True):
            assert torch.equal(generate(m, prompt, 6, u=u, temperature=WARM, graph=graph), want)


@pytest.mark.parametrize("amp", [False, True])
def test_draws_of_many_tokens_eager_captured_and_from_the_dense_model(dev, amp):
    m, g = model(dev), torch.Generator().manual_seed(11)
    prompt, u = torch.randint(0, 997, (3, 20), generator=g).to(dev), torch.rand(3, 40, generator=g).to(dev)
    lengths = torch.tensor([20, 7, 1])
    eager, captured = (generate(m, prompt, 40, lengths, u, amp=amp, graph=graph, temperature=WARM, top_p=0.95)
                       for graph in (False, True))
    assert torch.equal(eager, captured) and len(eager.unique()) > 60
    seq = torch.cat([prompt[0], eager[0]])[None]
    rows = []
    dec = Decoder(m, 1, amp=amp, graph=True, temperature=0.0)
    for n in (20, 21):
        dec.prefill(seq[:, :n])
        rows.append(dec.rows.clone())
    with torch.no_grad(), torch.autocast("cuda", torch.bfloat16, enabled=amp):  # up to 8 bits of keys and values
        want = m.hidden(seq[:, :21])[0, 19:].float()
    assert (torch.cat(rows).float() - want).norm() < 0.15 * want.norm()
