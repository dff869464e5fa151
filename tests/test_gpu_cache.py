"""The 8-bit cache, attention over it and the draw of a token on the GPU, against the 64-bit oracle."""
import numpy as np
import pytest
import torch

import cache_oracle as O
from paper_01_anti_decoy_pnfirtau_amd import KVCache, cached_attention, sample_tokens
from paper_01_anti_decoy_pnfirtau_amd.pnfirtau_attention import causal_gaussian_taps
from test_cache_cpu import CALLS, F64, filled

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def test_every_byte_and_scale_is_read_exactly(dev):
    """All 256 bytes under all scales that append writes."""
    cache = KVCache.new(1, 1, 16, 256 * 16, page=64, dtype=F32, device=dev)
    cache.k.copy_(torch.arange(256, device=dev).repeat(256).view(64, 1, 64, 16).to(torch.uint8))
    cache.v.copy_(torch.arange(256, device=dev).repeat(256).view(64, 1, 4, 16, 16).to(torch.uint8))
    e = torch.arange(256).view(64, 1, 4)
    cache.k_scale.copy_(e.to(torch.uint8)), cache.v_scale.copy_(e.to(torch.uint8))
    k, v = (F64(t)[0, 0] for t in cache.read(0, 4096, F32))
    val = np.concatenate([O.E4M3, [np.nan], -O.E4M3, [np.nan]])
    for s in range(27, 247):  # 448 * 2^120 is beyond fp32
        want = (val * 2.0 ** (s - 127)).astype(np.float32)
        assert np.array_equal(k[16 * s:16 * s + 16].ravel(), want.astype(np.float64), equal_nan=True)
        assert np.array_equal(v[16 * s:16 * s + 16].T.ravel(), want.astype(np.float64), equal_nan=True)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("calls", CALLS)
@pytest.mark.parametrize("d,K", [(8, 7), (20, 16), (16, None), (33, 3), (64, 7), (80, 7), (128, 7), (200, 7), (256, 5)])
def test_append_and_read(dev, dtype, calls, d, K):
    taps = None if K is None else causal_gaussian_taps(K) if K % 2 else torch.rand(2, K)
    cache, want = filled(2, 2, d, calls, taps, dtype, device=dev)
    start, N, counts = calls[-1]
    for b in range(2):
        n = start[b] + (N if counts is None else counts[b])
        for got, exact in zip(cache.read(0, cache.capacity, F32), want.dense()):
            assert np.array_equal(F64(got[b, :, :n]), exact[b, :, :n])
        for got, exact in zip(cache.read(i32([3, 9], dev), 20), want.dense()):
            lo = (3, 9)[b]
            assert np.array_equal(F64(got[b]), F64(torch.tensor(exact[b, :, lo:lo + 20]).to(dtype)))


def random_cache(B, H, d, lengths, page, dev, seed, max_len=None):
    g = torch.Generator(device=dev).manual_seed(seed)
    cache = KVCache.new(B, H, d, max_len or max(lengths), page=page, dtype=F32, device=dev)
    n = cache.table.numel()
    cache.table.copy_(torch.randperm(n, generator=g, device=dev).view_as(cache.table).int())
    D = cache.k.shape[3]
    for t, at in ((cache.k, torch.arange(D, device=dev)), (cache.v, torch.arange(D, device=dev)[:, None])):
        x = (torch.randn(t.shape, generator=g, device=dev) * 128).clamp_(-448, 448) * (at < d)
        t.copy_(x.to(torch.float8_e4m3fn).view(torch.uint8))
    for t in (cache.k_scale, cache.v_scale):
        t.copy_(torch.randint(118, 123, t.shape, generator=g, device=dev).to(torch.uint8))
    return cache


def check_attention(dev, B, H, G, d, N, starts, page=32, dtype=BF16, gamma=0.5, causal=True, counts=None, tau=0.1,
                    max_len=None, scale=None, seed=0):
    lengths = [s + N for s in starts]
    cache = random_cache(B, H, d, lengths, page, dev, seed, max_len)
    g = torch.Generator().manual_seed(seed + 1)
    q = torch.randn(B, N, H * G, d, generator=g).transpose(1, 2).to(dtype)
    o = cached_attention(q.to(dev), cache, i32(starts, dev), torch.tensor(tau, device=dev), scale=scale, gamma=gamma,
                         causal_mask=causal, counts=None if counts is None else i32(counts, dev))
    assert o.shape == q.shape and o.dtype == dtype and o.transpose(1, 2).is_contiguous()
    k, v = (F64(t) for t in cache.read(0, max(lengths), F32))
    want, tol = O.attend(F64(q), k, v, starts, tau, d ** -0.5 if scale is None else scale, gamma, causal, counts,
                         low=dtype == BF16)
    err = np.abs(F64(o) - want)
    assert np.isfinite(F64(o)).all() and (err <= tol).all(), float((err / tol).max())
    again = cached_attention(q.to(dev), cache, i32(starts, dev), torch.tensor(tau, device=dev), scale=scale, gamma=gamma,
                             causal_mask=causal, counts=None if counts is None else i32(counts, dev))
    assert torch.equal(o, again)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [16, 32, 64, 128, 8, 40, 80, 96, 112, 144, 200, 256])
def test_attention_head_sizes(dev, dtype, d):
    check_attention(dev, 2, 2, 1, d, 1, [0, 70], dtype=dtype)
    check_attention(dev, 2, 1, 3, d, 7, [130, 3], dtype=dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("starts,N,page", [([0], 1, 16), ([62, 63, 64, 65], 1, 16), ([255, 256, 0], 1, 64),
                                           ([700, 5, 1300, 511, 512], 1, 128), ([2047, 1], 2, 32), ([0, 40], 33, 16),
                                           ([300, 0], 65, 256)])
def test_attention_lengths(dev, dtype, starts, N, page):
    check_attention(dev, len(starts), 2, 2, 32, N, starts, page=page, dtype=dtype)
    check_attention(dev, len(starts), 1, 1, 64, N, starts, page=page, dtype=dtype, max_len=max(starts) + N + 1000)


@pytest.mark.parametrize("gamma,causal,tau,scale", [(None, True, 0.1, None), (0.5, False, 0.1, None), (2.0, True, -1.0, 0.5),
                                                    (0.5, True, 1e3, None), (0.5, True, 0.0, 1e-3), (0.5, True, 0.0, 50.0),
                                                    (None, True, 0.0, 1e5), (None, True, 0.0, 1e-6)])
def test_attention_settings(dev, gamma, causal, tau, scale):
    for dtype in (BF16, F32):
        check_attention(dev, 2, 1, 2, 64, 20, [600, 17], dtype=dtype, gamma=gamma, causal=causal, tau=tau, scale=scale)
    check_attention(dev, 3, 2, 1, 32, 9, [500, 3, 0], counts=[4, 9, 0], gamma=gamma, causal=causal, tau=tau, scale=scale)


def test_values_that_are_not_finite_stay_where_they_are_seen(dev):
    for dtype in (BF16, F32):
        cache = random_cache(1, 1, 16, [300], 16, dev, 0)
        k, v = (torch.rand(1, 1, 8, 16, device=dev) for _ in range(2))
        v[0, 0, 5, 3] = torch.inf
        cache.append(k, v, 280)
        q = torch.rand(1, 1, 8, 16, device=dev).to(dtype)
        o = cached_attention(q, cache, 280, torch.tensor(0.0, device=dev))
        assert o.isnan()[0, 0].nonzero().tolist() == [[5, 3], [6, 3], [7, 3]]
        cache.append(torch.full((1, 1, 1, 16), torch.nan, device=dev), k[:, :, :1], 288)
        o = cached_attention(q[:, :, :2], cache, 287, torch.tensor(0.0, device=dev))
        assert o[0, 0, 0].isnan().sum() == 1 and o[0, 0, 1].isnan().all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("K", [None, 7])
def test_append_of_what_is_not_finite(dev, dtype, K):
    taps = None if K is None else causal_gaussian_taps(K)
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(1, 2, 50, 24, generator=g).to(dtype) for _ in range(2))
    for t in (k, v):
        t[0, 0, 20, 3], t[0, 1, 21, 5], t[0, 0, 40, :], t[0, 1, 7, 1] = torch.inf, -torch.inf, torch.nan, torch.nan
    k[0, 1, 33, 2] = torch.finfo(dtype).max
    cache, want = KVCache.new(1, 2, 24, 50, page=16, dtype=dtype, device=dev), O.Cache(1, 2, 24, 64)
    for a, b in ((0, 37), (37, 38), (38, 50)):
        cache.append(k[:, :, a:b].to(dev), v[:, :, a:b].to(dev), a, taps=None if K is None else taps.to(dev))
        with np.errstate(invalid="ignore"):
            want.append(F64(k[:, :, a:b]), F64(v[:, :, a:b]), [a], None if K is None else F64(taps))
    with np.errstate(over="ignore"):  # fp32's largest rounds up to 2^128 in e4m3, infinity as fp32
        want = [x.astype(np.float32) for x in want.dense()]
    for got, exact in zip(cache.read(0, 50, F32), want):
        assert np.array_equal(got[0].cpu().numpy(), exact[0, :, :50], equal_nan=True)


def test_what_does_not_fit_is_left_alone(dev):
    cache, want = filled(2, 2, 20, CALLS[1], causal_gaussian_taps(7), F32, device=dev)
    before = [t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale, cache.raw)]
    k = torch.rand(2, 2, 3, 20, device=dev)
    cache.append(k, k, i32([-1, cache.capacity - 2], dev))
    same = lambda: [torch.equal(a, b) for a, b in  # noqa: E731
                    zip(before, (cache.k, cache.v, cache.k_scale, cache.v_scale, cache.raw))]
    assert all(same())
    o = cached_attention(k, cache, i32([-1, cache.capacity - 2], dev), torch.tensor(0.0, device=dev))
    assert o.isnan().all()
    cache.table[0, 1], cache.table[0, 2] = -1, cache.k.shape[0]
    cache.append(k, k, i32([40, 0], dev), counts=i32([3, 0], dev))
    assert same()[:4] == [True] * 4
    o = cached_attention(k, cache, i32([30, 30], dev), torch.tensor(-9.0, device=dev))
    assert o[0, :, 2].isnan().all() and o[0, :, :2].isfinite().all() and o[1].isfinite().all()
    got = cache.read(i32([30, -2], dev), 4)
    assert got[0][0].isnan().any(0).any(-1).tolist() == [False, False, True, True]
    assert got[1][1, :, :2].eq(0).all()
    assert cache.read(cache.capacity - 1, 3)[1][1, :, 1:].eq(0).all()


SETTINGS = [dict(), dict(temperature=0.0), dict(temperature=0.3, top_k=5), dict(top_p=0.7), dict(min_p=0.1),
            dict(top_k=20, top_p=0.5, min_p=0.01), dict(top_k=1), dict(min_p=2.0), dict(top_k=900, top_p=0.9),
            dict(temperature=7.0, top_p=0.999), dict(top_p=0.0)]


@pytest.mark.parametrize("setting", SETTINGS)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [1, 2, 101, 1000, 8191, 33278, 140001])
def test_sampling(dev, setting, dtype, V):
    g = torch.Generator().manual_seed(V)
    rows = 24 if V < 10000 else 10
    z = (torch.randn(rows, V, generator=g) * 2).to(dtype)
    z[3] = -torch.inf
    z[4, V // 2] = torch.nan
    z[5, V // 2:] = -torch.inf
    z[6, :] = torch.finfo(dtype).min
    z[7, V // 3] = z[7, V - 1] = torch.inf
    z[8] = z[8].round()  # many equal ones
    u = torch.rand(rows, generator=g)
    u[0], u[1] = 0.0, 1 - 2.0 ** -24
    want = [O.sample(F64(z[i]), float(u[i]), **setting) for i in range(rows)]
    got = sample_tokens(z.to(dev), u.to(dev), **setting).tolist()
    # fixed point rounds each weight by half a unit of 2^-42 or less of the largest
    assert all(a == b or near < V * 2.0 ** -42 for a, (b, near) in zip(got, want)), (got, want)
    wide = torch.full((rows, V + 3), 9.0, dtype=dtype)
    wide[:, 1:V + 1] = z
    each = {n: torch.full((rows,), x, device=dev) for n, x in setting.items() if n in ("top_k", "temperature")}
    rest = {n: x for n, x in setting.items() if n not in each}
    if "temperature" not in setting or setting["temperature"] in (0.0, 7.0):
        assert sample_tokens(wide.to(dev)[:, 1:V + 1], u.to(dev), **rest, **each).tolist() == got
