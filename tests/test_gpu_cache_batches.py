"""Attention over the 8-bit cache of more sequences than a wave has lanes, which then look after several each; and of a
sequence beside others against the same one alone."""
import ctypes

import numpy as np
import pytest
import torch

import cache_oracle as O
from paper_01_anti_decoy_pnfirtau_amd import KVCache, _lib, cached_attention
from test_cache_cpu import F64
from test_gpu_cache import BF16, F32, i32, random_cache

pytestmark = pytest.mark.gpu


def in_pieces(cache, Hq, N, dtype):
    """Whether such a call is cut, for which it needs a workspace."""
    k, at = cache.k, ctypes.c_void_p
    c = _lib.PnfxCache(at(k.data_ptr()), at(cache.v.data_ptr()), at(cache.k_scale.data_ptr()), at(cache.v_scale.data_ptr()),
                       None, at(cache.table.data_ptr()), cache.table.shape[1], cache.table.shape[0], k.shape[1],
                       cache.raw.shape[3], k.shape[3], k.shape[2], k.shape[0], cache.table.shape[1])
    return _lib.lib().pnfx_cached_attn_workspace_size(ctypes.byref(c), Hq, N, 1 if dtype == BF16 else 0) > 0


@pytest.mark.parametrize("dtype,d,N,max_len", [(BF16, 16, 1, 3000), (F32, 16, 1, 3000), (BF16, 16, 5, 2100), (BF16, 72, 256, 1100)])
@pytest.mark.parametrize("B", [64, 65, 130, 191])
def test_batches_in_pieces(dev, B, dtype, d, N, max_len):
    """Lengths of all kinds, sequences without tokens and ones that are refused among them."""
    cache = random_cache(B, 1, d, [max_len], 64, dev, B)
    assert in_pieces(cache, 2, N, dtype)
    cap, rng = cache.capacity, np.random.default_rng(B + N)
    start = rng.integers(0, cap - N + 1, B)
    start[::7] = rng.integers(0, 40, len(start[::7]))
    counts = rng.integers(0, 4, B).clip(max=N) if N > 1 else (rng.random(B) < 0.8).astype(np.int64)
    counts[[3, B - 1]] = N  # of many rows, two with all of them
    start[B - 1] = cap - N
    bad = np.zeros(B, dtype=bool)
    bad[[5, 20, B - 2]] = True
    start[bad], counts[bad] = (-1, cap, cap - N + 1), (1, 1, N)
    q = torch.randn(B, 2, N, d, generator=torch.Generator().manual_seed(N)).to(dtype)
    args = i32(start.tolist(), dev), torch.tensor(0.1, device=dev)
    o = cached_attention(q.to(dev), cache, *args, counts=i32(counts.tolist(), dev))
    k, v = (F64(t) for t in cache.read(0, cap, F32))
    want, tol = O.attend(F64(q), k, v, np.where(bad, 0, start), float(np.float32(0.1)), d ** -0.5, 0.5,
                         counts=np.where(bad, 0, counts), low=dtype == BF16)
    got = F64(o)
    for b in np.flatnonzero(bad):
        assert np.isnan(got[b, :, :counts[b]]).all() and (got[b, :, counts[b]:] == 0).all()
    assert (np.abs(got - want)[~bad] <= tol[~bad]).all(), float((np.abs(got - want) / tol)[~bad].max())
    assert all((got[b, :, counts[b]:] == 0).all() for b in range(B))
    same = cached_attention(q.to(dev), cache, *args, counts=i32(counts.tolist(), dev))
    assert torch.equal(same.nan_to_num(7.0), o.nan_to_num(7.0))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d,N,max_len", [(64, 1, 6000), (128, 7, 4000), (80, 256, 1500), (200, 3, 2000)])
def test_a_sequence_beside_others_and_alone(dev, dtype, d, N, max_len):
    """Not bit by bit: how its keys are cut into pieces goes by all lengths."""
    B = 6
    cache = random_cache(B, 2, d, [max_len], 64, dev, 1)
    start = [max_len - N, 0, 700, 63, max_len // 2, 3]
    q = torch.randn(B, 4, N, d, generator=torch.Generator().manual_seed(2)).to(dtype)
    tau = torch.tensor(0.1, device=dev)
    o = cached_attention(q.to(dev), cache, i32(start, dev), tau)
    k, v = (F64(t) for t in cache.read(0, max_len, F32))
    want, tol = O.attend(F64(q), k, v, start, float(np.float32(0.1)), d ** -0.5, 0.5, low=dtype == BF16)
    for b in range(B):
        alone = KVCache(cache.k, cache.v, cache.k_scale, cache.v_scale, cache.raw[b:b + 1], cache.table[b:b + 1])
        one = cached_attention(q[b:b + 1].to(dev), alone, start[b], tau)
        for x in (o[b:b + 1], one):
            assert (np.abs(F64(x) - want[b:b + 1]) <= tol[b:b + 1]).all()
