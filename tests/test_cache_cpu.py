"""The 8-bit cache, attention over it and the draw of a token on CPU tensors, against the 64-bit oracle; refusals."""
import numpy as np
import pytest
import torch

import cache_oracle as O
from paper_01_anti_decoy_pnfirtau_amd import KVCache, cached_attention, sample_tokens
from paper_01_anti_decoy_pnfirtau_amd.pnfirtau_attention import causal_gaussian_taps

F64 = lambda t: t.detach().double().cpu().numpy()  # noqa: E731


def filled(B, H, d, calls, taps, dtype, page=32, max_len=96, seed=0, device="cpu"):
    """A cache and the oracle's after `calls` of (start [B], N, counts or None)."""
    g = torch.Generator().manual_seed(seed)
    cache = KVCache.new(B, H, d, max_len, page=page, dtype=dtype, device=device)
    cache.table.copy_(torch.randperm(cache.table.numel(), generator=g).view_as(cache.table).int())
    want = O.Cache(B, H, d, cache.capacity)
    for start, N, counts in calls:
        size = torch.exp(torch.randn(B, 1, N, 1, generator=g) * 2)  # tokens of different sizes: scales that grow
        k, v = (torch.randn(B, N, H, d, generator=g).transpose(1, 2).mul(size).to(dtype) for _ in range(2))
        dev = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
        cache.append(k.to(device), v.to(device), dev(start), taps=None if taps is None else taps.to(device),
                     counts=dev(counts))
        want.append(F64(k), F64(v), start, None if taps is None else F64(taps), counts)
    return cache, want


CALLS = [[([0, 0], 5, None), ([5, 5], 1, None), ([6, 6], 31, None), ([37, 37], 1, [1, 0])],
         [([0, 0], 40, [40, 23]), ([40, 23], 17, [17, 9]), ([57, 32], 2, None)]]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("calls", CALLS)
@pytest.mark.parametrize("d,K", [(8, 7), (20, 16), (16, None), (33, 3)])
def test_append_and_read(dtype, calls, d, K):
    taps = None if K is None else causal_gaussian_taps(K) if K % 2 else torch.rand(2, K)
    cache, want = filled(2, 2, d, calls, taps, dtype)
    start, N, counts = calls[-1]
    for b in range(2):
        n = start[b] + (N if counts is None else counts[b])
        for got, exact in zip(cache.read(0, cache.capacity, torch.float32), want.dense()):
            assert np.array_equal(F64(got[b, :, :n]), exact[b, :, :n])


@pytest.mark.parametrize("gamma,causal,G,d", [(0.5, True, 1, 20), (None, True, 2, 16), (0.5, False, 3, 8)])
def test_attention(gamma, causal, G, d):
    cache, want = filled(2, 2, d, CALLS[1], causal_gaussian_taps(7), torch.float32)
    q = torch.randn(2, 2 * G, 2, d)
    got = cached_attention(q, cache, torch.tensor([57, 32]), torch.tensor(0.2), gamma=gamma, causal_mask=causal)
    o, tol = O.attend(F64(q), *want.dense(), [57, 32], 0.2, d ** -0.5, gamma, causal)
    assert (np.abs(F64(got) - o) <= tol + 2.0 ** -20 * np.abs(o).max()).all()


@pytest.mark.parametrize("setting", [dict(), dict(temperature=0.0), dict(temperature=0.3, top_k=5), dict(top_p=0.7),
                                     dict(min_p=0.1), dict(top_k=20, top_p=0.5, min_p=0.01), dict(top_k=1), dict(min_p=2.0)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sampling(setting, dtype):
    g = torch.Generator().manual_seed(3)
    z = (torch.randn(40, 101, generator=g) * 2).to(dtype)
    z[3] = -torch.inf
    z[4, 7] = torch.nan
    z[5, 50:] = -torch.inf
    z[6, :] = torch.finfo(dtype).min
    z[7, 9] = z[7, 80] = torch.inf
    u = torch.rand(40, generator=g)
    got = sample_tokens(z, u, **setting).tolist()
    assert got == [O.sample(F64(z[i]), float(u[i]), **setting)[0] for i in range(40)]
    each = {n: torch.full((40,), x) for n, x in setting.items()}
    assert sample_tokens(z, u, **each).tolist()[8:] == [O.sample(F64(z[i]), float(u[i]), **{
        n: x if n == "top_k" else float(np.float32(x)) for n, x in setting.items()})[0] for i in range(8, 40)]


def test_refusals():
    cache = KVCache.new(2, 2, 20, 64, page=32, dtype=torch.float32, device="cpu")
    k = torch.zeros(2, 2, 5, 20)
    with pytest.raises(ValueError):
        cache.append(k, k, 60)
    with pytest.raises(ValueError):
        cache.append(k, k, -1)
    with pytest.raises(ValueError):
        cache.append(k, k, torch.tensor([0, 60]))
    with pytest.raises(ValueError):
        cache.append(k, k[:, :1], 0)
    with pytest.raises(TypeError):
        cache.append(k, k, torch.tensor([0.0, 1.0]))
    with pytest.raises(ValueError):
        cache.append(k, k, torch.tensor([0, 1, 2]))
    with pytest.raises(RuntimeError, match="no gradients"):
        cache.append(k.clone().requires_grad_(), k, 0)
    with pytest.raises(ValueError):
        cached_attention(torch.zeros(2, 3, 1, 20), cache, 0, torch.tensor(0.0))
    with pytest.raises(RuntimeError, match="no gradients"):
        cached_attention(torch.zeros(2, 2, 1, 20), cache, 0, torch.tensor(0.0, requires_grad=True))
    cache.table[1, 1] = 99
    with pytest.raises(ValueError, match="page"):
        cache.append(k, k, 40)
    with pytest.raises(ValueError, match="page"):
        cached_attention(k[:, :, :1], cache, 40, torch.tensor(0.0))
    assert cache.read(30, 4)[0][1].isnan().any(0).any(-1).tolist() == [False, False, True, True]
    assert cache.read(62, 4)[0][0].eq(0).all()
    with pytest.raises(ValueError):
        KVCache.new(2, 2, 20, 64, page=24, device="cpu")
    with pytest.raises(ValueError):
        KVCache.new(2, 2, 257, 64, device="cpu")
    with pytest.raises(ValueError):
        KVCache(cache.k, cache.v[..., :8], cache.k_scale, cache.v_scale, cache.raw, cache.table)
    with pytest.raises(TypeError):
        KVCache(cache.k, cache.v, cache.k_scale, cache.v_scale, cache.raw, cache.table.long())
    z, u = torch.zeros(3, 7), torch.zeros(3)
    for bad in (dict(temperature=-1.0), dict(top_p=-0.1), dict(top_k=-2), dict(min_p=float("nan")),
                dict(top_k=torch.zeros(2, dtype=torch.int32))):
        with pytest.raises(ValueError):
            sample_tokens(z, u, **bad)
    with pytest.raises(TypeError):
        sample_tokens(z, u, top_k=torch.zeros(3))
    with pytest.raises(TypeError):
        sample_tokens(z.half(), u)
    with pytest.raises(ValueError):
        sample_tokens(z, u.double())
    with pytest.raises(ValueError):
        sample_tokens(torch.zeros(3, 0), u)


def test_values_that_are_not_finite_stay_where_they_are_seen():
    cache = KVCache.new(1, 1, 16, 32, page=16, dtype=torch.float32, device="cpu")
    k, v = torch.rand(1, 1, 8, 16), torch.rand(1, 1, 8, 16)
    v[0, 0, 5, 3] = torch.inf
    cache.append(k, v, 0)
    o = cached_attention(torch.rand(1, 1, 8, 16), cache, 0, torch.tensor(0.0))
    assert o.isnan()[0, 0].nonzero().tolist() == [[5, 3], [6, 3], [7, 3]]
    cache.append(torch.full((1, 1, 1, 16), torch.nan), v[:, :, :1], 8)
    o = cached_attention(torch.rand(1, 1, 2, 16), cache, 7, torch.tensor(0.0))
    assert o[0, 0, 0].isnan().sum() == 1 and o[0, 0, 1].isnan().all()
