"""Arguments of the 8-bit cache, attention over it and the draw that a call must not take for others, on CPU tensors."""
import pytest
import torch
from torch.autograd import forward_ad

from paper_01_anti_decoy_pnfirtau_amd import KVCache, _lib, cached_attention, sample_tokens
from test_cache_abi_cpu import append, attend, cache as described

TAU = torch.tensor(0.0)


def new(B=2, H=2, d=20, max_len=64, **kw):
    return KVCache.new(B, H, d, max_len, page=32, dtype=torch.float32, device="cpu", **kw)


def test_counts_and_starts_that_are_no_whole_numbers():
    cache, k = new(), torch.randn(2, 2, 5, 20)
    for counts in (3, 3.0, [3, 3]):
        with pytest.raises(TypeError, match="counts"):
            cache.append(k, k, 0, counts=counts)
        with pytest.raises(TypeError, match="counts"):
            cached_attention(k, cache, 0, TAU, counts=counts)
    for start in (1.5, 1.0, "1"):
        with pytest.raises(TypeError):
            cache.append(k, k, start)
        with pytest.raises(TypeError):
            cache.read(start, 3)
    assert not cache.k.any()


def test_starts_of_a_compiled_call():
    cache, same, k = new(), new(), torch.randn(2, 2, 1, 20)

    def step(cache, k, start):
        cache.append(k, k, start)
        return cached_attention(k, cache, start, TAU)

    compiled = torch.compile(step, backend="eager")
    for start in (3, 4, 5, 9):
        assert torch.equal(compiled(cache, k, start), step(same, k, start))


def test_tangents_and_taps_that_ask_for_a_gradient():
    cache, k = new(), torch.randn(2, 2, 3, 20)
    with pytest.raises(RuntimeError, match="no gradients"):
        cache.append(k, k, 0, taps=torch.ones(3, requires_grad=True))
    with forward_ad.dual_level(), torch.no_grad():
        dual = forward_ad.make_dual(k, k)
        tau, taps = (forward_ad.make_dual(t, torch.ones_like(t)) for t in (TAU, torch.ones(3)))
        for call in (lambda: cache.append(dual, k, 0), lambda: cache.append(k, dual, 0),
                     lambda: cache.append(k, k, 0, taps=taps), lambda: cached_attention(dual, cache, 0, TAU),
                     lambda: cached_attention(k, cache, 0, tau)):
            with pytest.raises(RuntimeError, match="no gradients"):
                call()
        cache.append(k, k, 0)  # without one
    with torch.no_grad(), pytest.raises(RuntimeError, match="no gradients"):
        torch.func.jvp(lambda q: cached_attention(q, cache, 0, TAU), (k,), (k,))
    with pytest.raises(RuntimeError, match="no gradients"):
        torch.func.grad(lambda q: cached_attention(q, cache, 0, TAU).sum())(k)


@pytest.mark.parametrize("B,H,max_len,kw", [
    (1, 1, 1 << 17, dict(page=1 << 17)), (1, 1, 64, dict(page=0)), (1, 1, 64, dict(page=-16)), (1, 1, 64, dict(page=8)),
    (1, 1, (1 << 30) + 1, {}), (2, 1 << 17, 1 << 17, {}), (1, 1 << 20, 16, {}), (1, 0, 16, {}), (1, 2, 0, {}),
    (1, 2, 64, dict(pages=0)), (1 << 24, 1, 16, dict(pages=1))], ids=str)
def test_caches_that_no_kernel_takes(B, H, max_len, kw):
    """Shapes alone are looked at: nothing is allocated."""
    with pytest.raises(ValueError, match="KVCache"):
        KVCache.new(B, H, 16, max_len, device="meta", **kw)


def test_the_largest_caches():
    assert KVCache.new(1, 1, 16, 1 << 16, device="meta", page=1 << 16).capacity == 1 << 16
    assert KVCache.new(1, 1, 16, 1 << 30, device="meta").capacity == 1 << 30
    KVCache.new(1, 2 ** 20 - 1, 16, 16, device="meta", page=16)
    KVCache.new(2 ** 24 - 1, 1, 16, 16, device="meta", page=16)
    KVCache.new(0, 2, 16, 16, device="meta")


def test_the_c_entry_names_both_ends_of_the_page_size():
    assert append(described(page=1 << 17)) != 0
    assert b"131072" in _lib.lib().pnfx_last_error() and b"16 to 65536" in _lib.lib().pnfx_last_error()


def test_numbers_of_blocks_and_rows_beyond_64_bits():
    """2 * 2^23 * 2^19 * 2^21 groups of blocks, 2^42 * 2^14 row tiles of 256 threads: both were 0 of 2^64."""
    c = described(B=1 << 23, H=1 << 19, pages=1)
    assert append(c, N=(1 << 26) - 30) != 0
    assert b"B=8388608 H=524288" in _lib.lib().pnfx_last_error()
    assert attend(c, Hq=1 << 19, N=1 << 19) != 0
    assert b"B=8388608 H=524288" in _lib.lib().pnfx_last_error()
    assert attend(described(B=1 << 12, H=1 << 18, pages=1), Hq=1 << 18, N=1 << 19) != 0
    assert b"row tiles in one call" in _lib.lib().pnfx_last_error()
    assert attend(described(), N=(1 << 31) - 200) != 0
    assert b"N=2147483448" in _lib.lib().pnfx_last_error()


def test_rows_without_scores_under_a_gamma_that_fp32_does_not_hold():
    cache, k = new(), torch.randn(2, 2, 5, 20)
    cache.append(k, k, 0)
    assert cached_attention(k, cache, 0, torch.tensor(1e9), gamma=1e-50).eq(0).all()
    want = cached_attention(k, cache, 0, TAU, gamma=None)
    assert torch.equal(cached_attention(k, cache, 0, TAU, gamma=1e-50), want)


def test_whole_numbers_of_more_than_32_bits():
    cache, k, far = new(), torch.randn(2, 2, 5, 20), 1 << 32
    with pytest.raises(ValueError, match="beside"):
        cache.append(k, k, torch.tensor([0, far + 3]))
    with pytest.raises(ValueError, match="beside"):
        cached_attention(k, cache, torch.tensor([0, -far]), TAU)
    cache.append(k, k, 0, counts=torch.tensor([far + 2, 5]))  # more than the call's: all of them
    assert cache.read(torch.tensor([0, far]), 5)[0][0].any(-1).all() and not cache.read(torch.tensor([0, far]), 5)[0][1].any()
    z, u = torch.randn(3, 50), torch.rand(3)
    every = sample_tokens(z, u).tolist()
    assert sample_tokens(z, u, top_k=torch.tensor([far + 1, far, 1 << 62])).tolist() == every
    assert sample_tokens(z, u, top_k=1 << 70).tolist() == every and sample_tokens(z, u, top_k=50.0).tolist() == every
    for k in (0.5, 2.5, float("inf")):
        with pytest.raises(ValueError, match="top_k"):
            sample_tokens(z, u, top_k=k)


@pytest.mark.parametrize("at", [0, -9, 64, 1 << 30])
def test_sequences_without_tokens_may_be_anywhere(at):
    """Of an empty cache, too, and of pages that do not exist; their rows are zeros."""
    cache, k = new(), torch.randn(2, 2, 5, 20)
    none, some = torch.tensor([0, 0]), torch.tensor([0, 5])
    cache.table[0, :] = -1
    start = torch.tensor([at, 0])
    cache.append(k, k, start, counts=none)
    assert cached_attention(k, cache, start, TAU, counts=none).eq(0).all() and not cache.k.any()
    cache.append(k, k, start, counts=some)
    for causal in (True, False):
        o = cached_attention(k, cache, start, TAU, counts=some, causal_mask=causal)
        alone = new(1)
        alone.append(k[1:], k[1:], 0)
        assert o[0].eq(0).all() and torch.equal(o[1:], cached_attention(k[1:], alone, 0, TAU, causal_mask=causal))
    with pytest.raises(ValueError):
        cached_attention(k, cache, start, TAU, counts=torch.tensor([1, 5]))


def test_random_numbers_and_settings_beside_their_range():
    """A token that is not kept is never drawn; what is no number is 0, or cuts nothing off."""
    z = torch.tensor([[-torch.inf, 1.0, 3.0, 2.0, -torch.inf, 0.0]]).repeat(5, 1)
    u = torch.tensor([1.0, 7.0, -0.5, float("nan"), 0.0])
    assert sample_tokens(z, u, top_k=2).tolist() == [3, 3, 2, 2, 2]
    assert sample_tokens(z, u).tolist() == [5, 5, 1, 1, 1]
    nan, u = torch.full((5,), float("nan")), torch.tensor([0.05, 0.3, 0.6, 0.9, 0.99])
    every = sample_tokens(z, u).tolist()
    assert sample_tokens(z, u, top_p=nan).tolist() == every and sample_tokens(z, u, min_p=nan).tolist() == every
    assert sample_tokens(z, u, temperature=nan).tolist() == [2] * 5


def test_tau_is_one_value():
    cache, k = new(), torch.randn(2, 2, 5, 20)
    cache.append(k, k, 0)
    want = cached_attention(k, cache, 0, TAU + 0.3)
    assert torch.equal(cached_attention(k, cache, 0, torch.full((1, 1, 1, 1, 1), 0.3)), want)
    for shape in (5, 2, 0, (2, 1, 1)):
        with pytest.raises(ValueError, match="score_tau"):
            cached_attention(k, cache, 0, torch.full((shape,) if isinstance(shape, int) else shape, 0.3))


def test_a_single_row_of_logits():
    z, u = torch.randn(40), torch.rand(1)
    want = sample_tokens(z[None], u, top_k=7, temperature=0.5)
    got = sample_tokens(z, u[0], top_k=torch.tensor(7), temperature=torch.tensor(0.5))
    assert got.shape == () and got == want[0]
    many = z.expand(5, 40)
    assert sample_tokens(many, u.expand(5), top_k=7, temperature=0.5).tolist() == want.tolist() * 5
    assert sample_tokens(many.t().contiguous().t(), u.expand(5), top_k=7, temperature=0.5).tolist() == want.tolist() * 5
