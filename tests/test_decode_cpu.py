"""Layers and the language model over the 8-bit cache, on CPU tensors: against the dense layers, and by pieces."""
import pytest
import torch

from paper_01_anti_decoy_pnfirtau_amd import PnFirConfig, PnFirTauFlashMHA, PnFirTauMHA, PnFirTauTritonMHA
from paper_01_anti_decoy_pnfirtau_amd.wikilm import Decoder, WikiLM, WikiLMConfig, generate


def model(**kw):
    torch.manual_seed(0)
    return WikiLM(97, WikiLMConfig(d_model=32, n_heads=2, n_layers=2, d_ff=48, max_seq=40, dropout=0.0, **kw),
                  "pn_fir_tau").eval()


def test_a_layer_over_the_cache_is_the_dense_layer_up_to_8_bits():
    torch.manual_seed(1)
    layer = PnFirTauMHA(PnFirConfig(d_model=64, n_heads=2)).eval()
    x = torch.randn(2, 30, 64)
    with torch.no_grad():
        want = layer(x)
        cache = layer.new_cache(2, 30, page=16)
        got = torch.cat([layer.forward_cached(x[:, a:b], cache, a) for a, b in ((0, 17), (17, 18), (18, 30))], 1)
    # keys and values are off by 2^-4 of themselves at most, a score by that of its terms' sum
    assert (got - want).norm() < 0.15 * want.norm()
    with torch.no_grad():  # the same cache, whatever the pieces, but for scales that grew: here one call
        one = layer.new_cache(2, 30, page=16)
        whole = layer.forward_cached(x, one, 0)
    assert (got - whole).norm() < 0.1 * want.norm()


def test_layers_that_have_no_cache():
    for kw in (dict(p=2.0), dict(silence_mode="mass_pow"), dict(causal_mask=False)):
        layer = PnFirTauMHA(PnFirConfig(d_model=32, n_heads=2, **kw))
        with torch.no_grad(), pytest.raises(ValueError):
            layer.forward_cached(torch.randn(1, 3, 32), layer.new_cache(1, 8, page=16), 0)
    layer = PnFirTauFlashMHA(PnFirConfig(d_model=32, n_heads=2, p=2.0))  # whose forward goes by p = 10 too
    with torch.no_grad():
        layer.forward_cached(torch.randn(1, 3, 32), layer.new_cache(1, 8, page=16), 0)


def test_generate_is_the_draw_from_the_model_over_its_cache():
    m = model()
    prompt = torch.randint(0, 97, (3, 9))
    lengths = torch.tensor([9, 4, 1])
    u = torch.rand(3, 6)
    got = generate(m, prompt, 6, lengths, u, temperature=0.7, top_k=30)
    for b in range(3):  # each by itself, unpadded
        alone = generate(m, prompt[b:b + 1, :lengths[b]], 6, u=u[b:b + 1], temperature=0.7, top_k=30)
        assert torch.equal(got[b:b + 1], alone)
    greedy = generate(m, prompt[:1], 5, temperature=0.0)
    with torch.no_grad():  # the first token: of the logits of the prompt's last row
        first = m.head(m.hidden_cached(prompt[:1], m.new_caches(1), 0)[:, -1]).argmax(-1)
    assert greedy[0, 0] == first[0]


def test_generate_refuses():
    m = model()
    prompt = torch.randint(0, 97, (1, 30))
    with pytest.raises(ValueError):
        generate(m, prompt, 11)  # more than max_seq
    with pytest.raises(ValueError):
        generate(m, prompt, 3, u=torch.rand(1, 2))
    with pytest.raises(ValueError):
        Decoder(model().train(), 1)
    dec = Decoder(m, 1, 32)
    with pytest.raises(ValueError):
        dec.prefill(torch.randint(0, 97, (2, 3)))
    dec.prefill(prompt)
    dec.step(torch.rand(1)), dec.step(torch.rand(1))
    with pytest.raises(ValueError):
        dec.step(torch.rand(1))


def test_weights_that_change_inside_the_caller_s_autocast():
    """A decoder's casts of the weights are its own: none is kept by a context around its calls."""
    m, prompt = model(), torch.randint(0, 97, (2, 9))
    with torch.autocast("cpu", torch.bfloat16):
        dec = Decoder(m, 2, amp=True, temperature=0.0)
        dec.prefill(prompt)
        before = dec.rows.clone()
        with torch.no_grad():
            m.blocks[0].attn.out.weight.mul_(-3), m.embed.weight.mul_(0.5)
        dec.prefill(prompt)
        got = [dec.rows.clone(), dec.step(torch.rand(2)).clone(), dec.rows.clone()]
    dec = Decoder(m, 2, amp=True, temperature=0.0)
    dec.prefill(prompt)
    want = [dec.rows.clone(), dec.step(torch.rand(2)).clone(), dec.rows.clone()]
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and not torch.equal(before, want[0])


def test_a_start_below_zero_is_refused_by_the_cache_not_met_by_the_embedding():
    m = model()
    with torch.no_grad(), pytest.raises(ValueError, match="append"):
        m.hidden_cached(torch.randint(0, 97, (2, 3)), m.new_caches(2), torch.tensor([-1, 3]))


def test_positions_that_the_model_does_not_have():
    m, idx = model(), torch.randint(0, 97, (2, 3))  # max_seq = 40, in pages of 64
    with pytest.raises(ValueError, match="new_caches"):
        m.new_caches(2, 41)
    with torch.no_grad():
        with pytest.raises(ValueError, match="hidden_cached"):
            m.hidden_cached(idx, m.new_caches(2), 38)
        assert m.hidden_cached(idx, m.new_caches(2), 37).isfinite().all()
        got = m.hidden_cached(idx, m.new_caches(2), torch.tensor([39, 4]))
        assert got[0, 0].isfinite().all() and got[0, 1:].isnan().all() and got[1].isfinite().all()
        got = m.hidden_cached(idx, m.new_caches(2), 38, counts=torch.tensor([2, 3]))
        assert got[:, :2].isfinite().all() and got[1, 2].isnan().all()


def test_steps_without_prompts_and_with_other_numbers_of_u():
    dec, prompt = Decoder(model(), 2, 12, temperature=0.0), torch.randint(0, 97, (2, 9))
    with pytest.raises(ValueError, match="prompts"):
        dec.step(torch.rand(2))
    dec.prefill(prompt)
    for u in (torch.rand(1), torch.rand(()), torch.rand(2, 1), torch.rand(3)):
        with pytest.raises(ValueError, match="u has shape"):
            dec.step(u)
    for _ in range(3):  # a refused step takes no room
        dec.step(torch.rand(2))


def test_lengths_outside_their_prompts():
    dec, prompt = Decoder(model(), 2, 12, temperature=0.0), torch.randint(0, 97, (2, 9))
    for lengths in ([9, 0], [10, 3], [-1, 2]):
        with pytest.raises(ValueError, match="lengths"):
            dec.prefill(prompt, torch.tensor(lengths))
    with pytest.raises(TypeError):
        dec.prefill(prompt, torch.tensor([9.0, 2.5]))
    with pytest.raises(TypeError):
        dec.prefill(prompt, 4)
    with pytest.raises(ValueError):
        dec.prefill(prompt, torch.tensor([9]))
    dec.prefill(prompt, torch.tensor([1, 9]))
    assert dec.step(torch.rand(2)).min() >= 0


@pytest.mark.parametrize("cls", [PnFirTauMHA, PnFirTauTritonMHA, PnFirTauFlashMHA])
def test_layers_that_have_a_cache_are_those_whose_forward_it_repeats(cls):
    def runs(**kw):
        layer = cls(PnFirConfig(d_model=32, n_heads=2, **kw))
        with torch.no_grad():
            try:
                layer.forward_cached(torch.randn(1, 3, 32), layer.new_cache(1, 8, page=16), 0)
            except ValueError:
                return False
        return True

    eager, rows = cls is PnFirTauMHA, cls is not PnFirTauFlashMHA
    assert runs(p=2.0) is not rows
    assert runs(silence_mode="mass_pow") is not eager
    for gamma in (None, 0.0, -1.0):  # no gate
        assert runs(silence_mode="mass_pow", silence_gamma=gamma)
