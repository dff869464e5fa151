"""What the C entry points of the 8-bit cache and of the draw refuse, and the workspace's size: no GPU is reached."""
import ctypes

import pytest
import torch

from paper_01_anti_decoy_pnfirtau_amd import KVCache, _lib, cached_attention, sample_tokens

P, ODD = 256, 264
F32, BF16 = 0, 1
GOOD = dict(k=P, v=P, k_scale=P, v_scale=P, raw=P, table=P, table_rs=4, B=2, H=2, d=20, D=32, page=64, pages=8, width=4)
BAD_CACHES = [dict(k=0), dict(v=0), dict(k_scale=0), dict(v_scale=0), dict(table=0), dict(k=ODD), dict(v=ODD), dict(B=0),
              dict(H=0), dict(pages=0), dict(width=0), dict(d=0), dict(d=257, D=272), dict(D=20), dict(D=48),
              dict(page=24), dict(page=8), dict(page=1 << 17), dict(table_rs=3), dict(B=1 << 24), dict(pages=1 << 31),
              dict(pages=1 << 30), dict(width=1 << 31, table_rs=1 << 31), dict(width=1 << 25, table_rs=1 << 25)]


def cache(**kw):
    return ctypes.byref(_lib.PnfxCache(**{**GOOD, **kw}))


def append(c, k=P, v=P, N=3, start=None, start_all=0, taps=None, taps_rows=1, K=7, dtype=F32):
    return _lib.lib().pnfx_cache_append(c, k, 0, 0, 20, v, 0, 0, 20, N, start, start_all, None, taps, taps_rows, K, dtype, None)


def read(c, k=P, v=P, first=0, count=3, dtype=F32):
    return _lib.lib().pnfx_cache_read(c, None, first, count, k, v, dtype, None)


def attend(c, q=P, o=P, tau=P, Hq=2, N=1, start=0, dtype=F32, ws=P, wsb=0):
    return _lib.lib().pnfx_cached_attn(c, q, 0, 20, 20, o, 0, 20, 20, Hq, N, None, start, None, tau, 1.0, 0.5, 1, 1, dtype,
                                       ws, wsb, None)


@pytest.mark.parametrize("bad", BAD_CACHES, ids=str)
def test_caches_that_no_kernel_may_see(bad):
    lib = _lib.lib()
    for call, name in ((append, b"cache_append"), (read, b"cache_read"), (attend, b"cached_attn")):
        assert call(cache(**bad)) != 0
        assert lib.pnfx_last_error().startswith(name)
    assert lib.pnfx_cached_attn_workspace_size(cache(**bad), 2, 1, BF16) == 0


def test_null_caches():
    for call in (append, read, attend):
        assert call(None) != 0
    assert _lib.lib().pnfx_cached_attn_workspace_size(None, 2, 1, BF16) == 0


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=None), dict(N=0), dict(N=-1), dict(N=1 << 31), dict(start_all=-1),
                                 dict(start_all=1 << 31), dict(taps=P, K=0), dict(taps=P, K=17),
                                 dict(taps=P, taps_rows=3), dict(taps=P, taps_rows=0), dict(dtype=2)], ids=str)
def test_append_refuses(bad):
    assert append(cache(), **bad) != 0


def test_append_needs_raw_keys_for_a_fir_and_a_grid_that_fits():
    assert append(cache(raw=None), taps=P) != 0
    assert append(cache(B=(1 << 24) - 1, H=64), N=1 << 20) != 0


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=None), dict(first=-1), dict(first=1 << 31), dict(count=0),
                                 dict(count=1 << 31), dict(dtype=7)], ids=str)
def test_read_refuses(bad):
    assert read(cache(), **bad) != 0


@pytest.mark.parametrize("bad", [dict(q=None), dict(o=None), dict(tau=None), dict(Hq=1), dict(Hq=3), dict(Hq=1 << 20),
                                 dict(N=0), dict(N=1 << 31), dict(start=-1), dict(start=1 << 31), dict(dtype=-1)], ids=str)
def test_attention_refuses(bad):
    assert attend(cache(), **bad) != 0


def test_attention_needs_its_workspace():
    lib, long = _lib.lib(), dict(width=512, table_rs=512)
    need = lib.pnfx_cached_attn_workspace_size(cache(**long), 2, 1, BF16)
    # two units (a sequence's key head each), at most the card's slots more pieces of one row of 32 columns each
    assert 0 < need < 64 << 20
    for ws, wsb in ((None, need), (P, need - 1), (ODD, need)):
        assert attend(cache(**long), dtype=BF16, ws=ws, wsb=wsb) != 0
        assert b"workspace" in lib.pnfx_last_error()
    assert lib.pnfx_cached_attn_workspace_size(cache(**long), 3, 1, BF16) == 0
    assert lib.pnfx_cached_attn_workspace_size(cache(**long), 2, 0, BF16) == 0


@pytest.mark.parametrize("bad", [dict(z=None), dict(u=None), dict(tokens=None), dict(settings=None), dict(B=0),
                                 dict(B=1 << 22), dict(V=0), dict(V=(1 << 20) + 1), dict(rs=6), dict(dtype=3)], ids=str)
def test_draw_refuses(bad):
    a = {**dict(z=P, rs=7, B=2, V=7, u=P, settings=ctypes.byref(_lib.PnfxSampling(1.0, 1.0, 0.0, 0)), tokens=P, dtype=F32),
         **bad}
    if a["V"] > 7:
        a["rs"] = a["V"]
    assert _lib.lib().pnfx_sample(*a.values(), None) != 0
    assert _lib.lib().pnfx_last_error().startswith(b"sample")


def test_empty_calls_and_other_head_sizes_on_the_cpu():
    c = KVCache.new(2, 2, 20, 64, page=32, dtype=torch.float32, device="cpu")
    k, none, tau = torch.randn(2, 2, 4, 20), torch.zeros(2, 2, 0, 20), torch.tensor(0.0)
    c.append(k, k, 0)
    before = c.read(0, 64)
    c.append(none, none, 3)
    c.append(k, k, 2, counts=torch.tensor([0, 0]))
    assert all(torch.equal(a, b) for a, b in zip(before, c.read(0, 64)))
    assert cached_attention(none, c, 3, tau).shape == (2, 2, 0, 20)
    assert [t.shape for t in c.read(3, 0)] == [(2, 2, 0, 20)] * 2
    with pytest.raises(ValueError, match="head size"):
        cached_attention(torch.zeros(2, 2, 1, 25), c, 0, tau)  # rows of 32, too
    with pytest.raises(ValueError):
        c.read(0, -1)
    assert sample_tokens(torch.zeros(0, 7), torch.zeros(0)).shape == (0,)
    assert sample_tokens(torch.zeros(2, 0, 7), torch.zeros(2, 0)).shape == (2, 0)
    none = KVCache.new(0, 2, 20, 64, page=32, dtype=torch.float32, device="cpu", pages=1)
    none.append(k[:0], k[:0], 0)
    assert cached_attention(k[:0], none, 0, tau).shape == (0, 2, 4, 20)
