"""Attention over the 8-bit cache: many query rows, where the waves of a workgroup share their keys, and long contexts in
pieces at every head size."""
import pytest
import torch

from paper_01_anti_decoy_pnfirtau_amd import KVCache, cached_attention
from test_gpu_cache import BF16, F32, check_attention, i32, random_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [65, 72, 80, 96, 104, 112, 128])
def test_pieces_by_head_size(dev, d):
    check_attention(dev, 2, 1, 2, d, 131, [600, 3], page=64)


@pytest.mark.parametrize("starts,N,G,page", [([0], 600, 1, 16), ([513], 256, 1, 32), ([300, 0, 700], 86, 3, 64),
                                             ([2000, 64], 257, 1, 128), ([515, 511], 33, 8, 16)])
def test_pieces_by_length(dev, starts, N, G, page):
    check_attention(dev, len(starts), 2, G, 72, N, starts, page=page, max_len=max(starts) + N + 100)


@pytest.mark.parametrize("gamma,causal,tau,scale", [(None, True, 0.1, None), (0.5, False, 0.1, None), (2.0, True, -1.0, 0.5),
                                                    (0.5, True, 1e3, None), (0.5, True, 0.0, 50.0), (None, True, 0.0, 1e-6)])
def test_settings_and_counts(dev, gamma, causal, tau, scale):
    check_attention(dev, 4, 1, 1, 80, 300, [400, 17, 0, 250], counts=[300, 0, 129, 1], gamma=gamma, causal=causal, tau=tau,
                    scale=scale)


def test_workgroups_of_whole_units(dev):
    check_attention(dev, 32, 4, 1, 72, 256, [(7 * b) % 200 for b in range(32)], page=64, max_len=480)  # short contexts
    check_attention(dev, 64, 4, 1, 16, 256, [(5 * b) % 100 for b in range(64)], page=64, max_len=400,
                    counts=[(37 * b) % 257 for b in range(64)])
    check_attention(dev, 64, 8, 1, 72, 256, [(11 * b) % 300 for b in range(64)], page=64, max_len=600)  # longer ones


@pytest.mark.parametrize("B,cap", [(1, 700), (32, 300)])
def test_refused_sequences_missing_pages_and_strange_values(dev, B, cap):
    """One piece of a unit and the whole of it: what is not finite is seen from its position on, and nowhere before."""
    H, d, N = 8, 72, 256
    cache = KVCache.new(B + 2, H, d, cap, page=16, dtype=BF16, device=dev)
    g = torch.Generator(device=dev).manual_seed(3)
    k, v = (torch.rand(B + 2, H, N, d, generator=g, device=dev).to(BF16) for _ in range(2))
    cache.append(k, v, 10)
    bad = v.clone()
    bad[0, 1, 100, 5], bad[0, 1, 200, 71] = torch.inf, torch.nan
    cache.append(k[:, :, :10], v[:, :, :10], 0), cache.append(k, bad, 10)
    q, tau = torch.rand(B + 2, H, N, d, generator=g, device=dev).to(BF16), torch.zeros(1, device=dev)
    o = cached_attention(q, cache, 10, tau)
    for h, column, first in ((1, 5, 100), (1, 71, 200)):
        assert o[0, h, :first, column].isfinite().all() and o[0, h, first:, column].isnan().all()
    assert o.isnan().sum() == 156 + 56
    start = torch.full((B + 2,), 10, dtype=torch.int32, device=dev)
    start[-1], start[-2] = -1, cache.capacity - N + 1
    cache.table[-3, 3] = -1  # tokens 48 .. 63
    last = cached_attention(q, cache, start, tau, counts=torch.full_like(start, N))
    assert last[-2:].isnan().all()
    assert last[-3, :, :38].isnan().sum() == 0 and last[-3, :, 38:].isnan().all()
    if B > 1:
        assert torch.equal(last[:-3].nan_to_num(7.0), o[:-3].nan_to_num(7.0))
    nothing = cached_attention(q, cache, start, tau, counts=torch.zeros_like(start))
    assert nothing[:-2].eq(0).all()


def test_query_strides_and_a_captured_graph(dev):
    B, H, d, N = 2, 2, 80, 150
    cache = random_cache(B, H, d, [900, 700], 64, dev, 5)
    g = torch.Generator(device=dev).manual_seed(1)
    wide = torch.randn(B, N, 2 * H, d + 3, generator=g, device=dev).to(BF16)
    tau = torch.full((1,), 0.1, device=dev)
    q = wide[..., 1:d + 1].transpose(1, 2)  # rows that begin anywhere
    start, counts = i32([750, 500], dev), i32([150, 149], dev)
    want = cached_attention(q.contiguous(), cache, start, tau, counts=counts)
    assert torch.equal(cached_attention(q, cache, start, tau, counts=counts), want)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cached_attention(q, cache, start, tau, counts=counts)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        o = cached_attention(q, cache, start, tau, counts=counts)
    for s in ([750, 500], [10, 0], [300, 549]):
        start.copy_(i32(s, dev))
        graph.replay()
        assert torch.equal(o, cached_attention(q, cache, start, tau, counts=counts))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [7, 16, 40, 64, 100, 128, 144, 200, 256])
def test_long_contexts_in_pieces(dev, dtype, d):
    check_attention(dev, 2, 2, 2, d, 1, [700, 2900], dtype=dtype, page=64)
    check_attention(dev, 2, 1, 3, d, 9, [1500, 3], dtype=dtype, page=16, counts=[9, 4])
