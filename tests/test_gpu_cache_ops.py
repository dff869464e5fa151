"""The 8-bit cache's operators as callers use them: operator checks, compiled, captured, on other streams, with other
strides and types of arguments, shared pages, caches beyond 2^32 bytes; what stays as it was."""
import numpy as np
import pytest
import torch

import cache_oracle as O
from paper_01_anti_decoy_pnfirtau_amd import KVCache, cached_attention, sample_tokens
from paper_01_anti_decoy_pnfirtau_amd.pnfirtau_attention import causal_gaussian_taps
from test_cache_cpu import CALLS, F64, filled
from test_gpu_cache import BF16, F32, i32, random_cache

pytestmark = pytest.mark.gpu


def tensors(cache):
    return [cache.k, cache.v, cache.k_scale, cache.v_scale, cache.raw]


def tau(dev):
    return torch.tensor(0.1, device=dev)


def test_opcheck(dev):
    import paper_01_anti_decoy_pnfirtau_amd.ops  # noqa: F401

    P = torch.ops.pnfx
    cache = random_cache(2, 2, 20, [70, 70], 32, dev, 0)
    k = torch.randn(2, 2, 5, 20, device=dev)
    start, taps = i32([60, 3], dev), causal_gaussian_taps(7).to(dev)
    c = (cache.k, cache.v, cache.k_scale, cache.v_scale)
    torch.library.opcheck(P.cache_append.default, (k, k, *c, cache.raw, cache.table, start, 0, None, taps))
    torch.library.opcheck(P.cache_read.default, (*c, cache.table, start, 0, 7, 20, BF16))
    torch.library.opcheck(P.cached_attn.default, (k, *c, cache.table, None, 50, i32([5, 2], dev), tau(dev), 0.2, 0.5, True, True))
    z, u = torch.randn(3, 50, device=dev), torch.rand(3, device=dev)
    torch.library.opcheck(P.sample_tokens.default, (z, u, 0.7, 5, 0.9, 0.0, None, i32([1, 2, 3], dev), None, None))


def test_compiled(dev):
    cache, same = (filled(2, 2, 20, CALLS[1], causal_gaussian_taps(7), F32, device=dev)[0] for _ in range(2))
    taps, q, u = causal_gaussian_taps(7).to(dev), torch.randn(2, 2, 1, 20, device=dev), torch.rand(2, device=dev)

    t0 = tau(dev)

    def step(cache, q, start):
        cache.append(q, q * 2, start, taps=taps)
        o = cached_attention(q, cache, start, t0)
        return o, sample_tokens(o[:, 0, 0], u, top_k=3)

    start = i32([59, 34], dev)
    got = torch.compile(step, fullgraph=True)(cache, q, start)
    want = step(same, q, start)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(torch.equal(a, b) for a, b in zip(tensors(cache), tensors(same)))


def test_captured_graphs_move_on_with_start(dev):
    """Two captured steps over caches of their own, replayed in turn with eager work and waits between, against an
    eager run of each."""
    taps, t0 = causal_gaussian_taps(7).to(dev), tau(dev)
    g = torch.Generator(device=dev).manual_seed(0)
    q, k, v = (torch.randn(2, 30, 3, 2, 1, 32, generator=g, device=dev) for _ in range(3))  # [graph, step, B, H, 1, d]

    def run(cache, start, q, k, v):
        cache.append(k, v, start, taps=taps)
        return cached_attention(q, cache, start, t0)

    want = []
    for i in range(2):
        cache, start = KVCache.new(3, 2, 32, 700, page=16, dtype=F32, device=dev), i32([0, 500, 17], dev)
        want.append([run(cache, start + t, q[i, t], k[i, t], v[i, t]) for t in range(30)])
    graphs = []
    for i in range(2):
        cache, start = KVCache.new(3, 2, 32, 700, page=16, dtype=F32, device=dev), i32([0, 500, 17], dev)
        box = [torch.zeros_like(q[0, 0]) for _ in range(3)]
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            run(cache, start, *box)  # a first call outside the capture; its token is written again by the replay
            for t in tensors(cache):
                t.zero_()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = run(cache, start, *box)
            start += 1
        graphs.append((graph, box, o, cache, start))  # which the graph's calls go on using
    for t in range(30):
        for i in (0, 1) if t % 2 else (1, 0):
            graph, box, o = graphs[i][:3]
            for b, x in zip(box, (q, k, v)):
                b.copy_(x[i, t])
            graph.replay()
            assert torch.equal(o, want[i][t])
        torch.cuda.synchronize()


def test_other_streams_and_threads(dev):
    import threading

    taps, out = causal_gaussian_taps(7).to(dev), {}

    def work(i, stream):
        with torch.cuda.device(dev), torch.cuda.stream(stream):
            cache, _ = filled(2, 2, 64, CALLS[1], taps.cpu(), BF16, device=dev, seed=i)
            q = torch.randn(2, 4, 2, 64, generator=torch.Generator().manual_seed(i)).to(dev, BF16)
            o = [cached_attention(q, cache, i32([57, 32], dev), tau(dev)) for _ in range(20)]
            z = torch.randn(5, 40000, generator=torch.Generator().manual_seed(i)).to(dev)
            s = [sample_tokens(z, torch.full((5,), 0.3, device=dev), top_p=0.8) for _ in range(20)]
            stream.synchronize()
            out[i] = o, s

    ref = {}
    for i in range(4):
        work(i, torch.cuda.current_stream())
        ref[i] = out[i]
    threads = [threading.Thread(target=work, args=(i, torch.cuda.Stream())) for i in range(4)]
    [t.start() for t in threads], [t.join() for t in threads]
    for i in range(4):
        for a, b in zip(ref[i][0] + ref[i][1], out[i][0] + out[i][1]):
            assert torch.equal(a, b)


@pytest.mark.parametrize("d", [20, 64, 128, 200])
def test_strides_and_forms_of_arguments(dev, d):
    taps = causal_gaussian_taps(7).to(dev)
    g = torch.Generator(device=dev).manual_seed(0)
    rows = torch.randn(2, 9, 3 * 2 * d + 5, generator=g, device=dev).to(BF16)
    q, k, v = (rows[..., i * 2 * d:(i + 1) * 2 * d].unflatten(2, (2, d)).transpose(1, 2) for i in range(3))  # odd rows
    forms = {
        "plain": (q.contiguous(), k.contiguous(), v.contiguous()),
        "rows": (q, k, v),
        "columns": tuple(t.transpose(2, 3).contiguous().transpose(2, 3) for t in (q, k, v)),
        "shared": (q, k[:, :1].expand(-1, 2, -1, -1), v[:1].expand(2, -1, -1, -1)),
    }
    got = {}
    for name, (a, b, c) in forms.items():
        for start in (i32([30, 30], dev), torch.tensor([30, 30], device=dev), 30):
            cache = random_cache(2, 2, d, [60, 60], 32, dev, 1)
            cache.raw = torch.zeros(2, 2, 16, d, dtype=BF16, device=dev)
            cache.append(b, c, start, taps=taps if name != "columns" else taps.expand(2, 7))
            o = cached_attention(a, cache, start, tau(dev))
            got.setdefault(name, []).append((o, *tensors(cache)))
    for name, each in got.items():
        same = "plain" if name != "shared" else "shared"
        for x in each:
            assert all(torch.equal(s, t) for s, t in zip(x, got[same][0]))
    a, b, c = (t.contiguous() for t in forms["shared"])
    cache = random_cache(2, 2, d, [60, 60], 32, dev, 1)
    cache.raw = torch.zeros(2, 2, 16, d, dtype=BF16, device=dev)
    cache.append(b, c, 30, taps=taps)
    assert all(torch.equal(s, t) for s, t in zip(tensors(cache), got["shared"][0][1:]))


def test_only_the_call_s_tokens_change(dev):
    cache = random_cache(2, 2, 40, [200, 200], 64, dev, 2)
    before = [t.clone() for t in tensors(cache)]
    new = torch.randn(2, 2, 30, 40, device=dev) * 0.01  # no scale grows
    cache.append(new, new, i32([37, 64], dev), counts=i32([30, 0], dev))
    pos = torch.arange(256, device=dev)
    page, place = cache.table.long()[:, pos // 64], pos % 64
    for b in range(2):
        mine = (pos >= 37) & (pos < 67) & (b == 0)
        for h in range(2):
            for t in range(256):
                a = [x[page[b, t], h, place[t]] for x in (before[0], cache.k)]
                c = [x[page[b, t], h, place[t] // 16, :, place[t] % 16] for x in (before[1], cache.v)]
                if not mine[t] and not (b == 0 and 32 <= t < 37):
                    assert torch.equal(*a) and torch.equal(*c)
    blocks = pos[::16]
    for x, y in ((before[2], cache.k_scale), (before[3], cache.v_scale)):
        same = (x == y).transpose(1, 2)[page[:, ::16], place[::16] // 16].all(2)  # [B, blocks]
        assert same[1].all() and same[0][(blocks + 15 < 48) | (blocks > 66)].all()
    assert torch.equal(before[4][1], cache.raw[1])


def test_shared_pages(dev):
    """Sequences with a common beginning: the pages are named twice, read alike, and each goes on in its own."""
    cache = random_cache(3, 2, 64, [300, 300, 300], 64, dev, 3)
    cache.table[1, :4], cache.table[2, :4] = cache.table[0, :4], cache.table[0, :4]
    q = torch.randn(1, 2, 1, 64, device=dev).expand(3, -1, -1, -1)
    o = cached_attention(q, cache, 255, tau(dev))
    assert torch.equal(o[0], o[1]) and torch.equal(o[0], o[2])
    k = torch.randn(3, 2, 4, 64, device=dev)
    cache.append(k, k, 256)
    o = cached_attention(q, cache, 259, tau(dev))
    for b in range(3):
        alone = KVCache(cache.k, cache.v, cache.k_scale, cache.v_scale, cache.raw[b:b + 1], cache.table[b:b + 1].clone())
        kv = [F64(t) for t in alone.read(0, 260, F32)]
        want, tol = O.attend(F64(q[b:b + 1]), *kv, [259], 0.1, 0.125, 0.5)
        assert (np.abs(F64(o[b:b + 1]) - want) <= tol).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("ke,ve,size", [(27, 127, 2.0 ** 104), (246, 127, 2.0 ** -115), (127, 27, 16.0), (127, 207, 16.0)])
def test_attention_at_the_ends_of_the_scales(dev, dtype, ke, ve, size):
    cache = random_cache(1, 2, 64, [90], 32, dev, 4)
    cache.k.copy_(cache.k & 0xb7)  # numbers below 1, so that values under the largest scale stay in fp32
    cache.k_scale.fill_(ke), cache.v_scale.fill_(ve)
    q = (torch.randn(1, 2, 3, 64, generator=torch.Generator().manual_seed(0)) * size).to(dtype)
    o = cached_attention(q.to(dev), cache, 87, tau(dev))
    k, v = (F64(t) for t in cache.read(0, 90, F32))
    want, tol = O.attend(F64(q), k, v, [87], float(np.float32(0.1)), 0.125, 0.5, low=dtype == BF16)
    assert np.isfinite(want).all() and np.abs(want).max() > 0
    assert (np.abs(F64(o) - want) <= tol).all()


def test_never_written_blocks_behind_a_sequence_do_not_reach_it(dev):
    for dtype in (F32, BF16):
        for byte in (0, 127, 255):
            cache = random_cache(1, 1, 64, [64], 64, dev, 5)
            q = torch.randn(1, 1, 1, 64, generator=torch.Generator().manual_seed(1)).to(dev, dtype)
            want = cached_attention(q, cache, 18, tau(dev))
            cache.k.view(-1, 16, 64)[2:], cache.v.view(-1, 64, 16)[2:] = byte, byte
            cache.k.view(-1, 16, 64)[1, 3:], cache.v.view(-1, 64, 16)[1, :, 3:] = byte, byte
            cache.k_scale[..., 2:], cache.v_scale[..., 2:] = byte, byte
            assert torch.equal(cached_attention(q, cache, 18, tau(dev)), want) and want.isfinite().all()


def test_beyond_32_bits_of_offset(dev):
    """4.4 GB of keys and as many values, a sequence in the last pages."""
    B, H, d, page, pages = 1, 1, 256, 1024, 17000
    table = torch.tensor([[pages - 1, 3, pages - 2]], dtype=torch.int32, device=dev)
    cache = KVCache.new(B, H, d, 3 * page, page=page, dtype=BF16, device=dev, pages=pages, table=table)
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(B, H, 3 * page, d, generator=g).to(BF16) for _ in range(2))
    cache.append(k.to(dev), v.to(dev), 0)
    small = KVCache.new(B, H, d, 3 * page, page=64, dtype=BF16, device=dev)
    small.append(k.to(dev), v.to(dev), 0)
    for a, b in zip(cache.read(0, 3 * page), small.read(0, 3 * page)):
        assert torch.equal(a, b) and a.abs().max() > 1
    q = torch.randn(B, 2, 2, d, generator=g).to(BF16).to(dev)
    a, b = (cached_attention(q, c, 3 * page - 2, tau(dev)) for c in (cache, small))
    assert torch.equal(a, b) and a.abs().max() > 0


def test_empty_calls(dev):
    cache = random_cache(2, 2, 20, [50, 50], 16, dev, 6)
    before = [t.clone() for t in tensors(cache)]
    none = torch.zeros(2, 2, 0, 20, device=dev)
    cache.append(none, none, 3)
    k = torch.randn(2, 2, 4, 20, device=dev)
    cache.append(k, k, i32([3, 9], dev), counts=i32([0, 0], dev))
    cache.append(k, k, i32([3, 9], dev), counts=i32([-3, 0], dev))
    assert all(torch.equal(a, b) for a, b in zip(before, tensors(cache)))
    assert cached_attention(none, cache, 3, tau(dev)).shape == (2, 2, 0, 20)
    assert cached_attention(k, cache, 3, tau(dev), counts=i32([0, 2], dev))[0].eq(0).all()
    assert [t.shape for t in cache.read(3, 0)] == [(2, 2, 0, 20)] * 2
    assert sample_tokens(torch.zeros(0, 7, device=dev), torch.zeros(0, device=dev)).shape == (0,)
    assert sample_tokens(torch.zeros(2, 0, 7, device=dev), torch.zeros(2, 0, device=dev)).shape == (2, 0)


def test_refusals(dev):
    cache = random_cache(2, 2, 20, [50, 50], 16, dev, 7)
    k = torch.randn(2, 2, 4, 20, device=dev)
    for call, error in (
            (lambda: cache.append(k, k, 47 + 16), ValueError),
            (lambda: cache.append(k, k[:, :, :3], 0), ValueError),
            (lambda: cache.append(k.to(BF16), k.to(BF16), 0), TypeError),
            (lambda: cache.append(k.half(), k.half(), 0), TypeError),
            (lambda: cache.append(k[:1], k[:1], 0), ValueError),
            (lambda: cache.append(k.cpu(), k.cpu(), 0), (ValueError, RuntimeError)),
            (lambda: cache.append(k, k, 0, taps=torch.ones(17, device=dev)), (ValueError, RuntimeError)),
            (lambda: cache.append(k, k, 0, taps=torch.ones(3, 7, device=dev)), (ValueError, RuntimeError)),
            (lambda: cache.append(k, k, i32([0, 0], "cpu")), ValueError),
            (lambda: cached_attention(k[:, :1], cache, 0, tau(dev)), ValueError),
            (lambda: cached_attention(k[..., :8], cache, 0, tau(dev)), ValueError),
            (lambda: cached_attention(k.half(), cache, 0, tau(dev)), TypeError),
            (lambda: cached_attention(k, cache, 0, torch.zeros(2, device=dev)), ValueError),
            (lambda: cached_attention(k, cache, 0, torch.zeros(1, device=dev, requires_grad=True)), RuntimeError),
            (lambda: cached_attention(k, cache, 0, tau(dev), counts=i32([1], dev)), ValueError),
            (lambda: cache.read(-1, 4), ValueError),
            (lambda: cache.read(0, 4, torch.float16), TypeError),
            (lambda: sample_tokens(torch.zeros(2, 7, device=dev), torch.zeros(2)), ValueError),
            (lambda: sample_tokens(torch.zeros(2, 1 << 20 | 1, device=dev, dtype=BF16), torch.zeros(2, device=dev)), ValueError)):
        with pytest.raises(error):
            call()


@pytest.mark.parametrize("dtype,V", [(F32, 1 << 20), (BF16, 1 << 20), (BF16, 12289), (BF16, 12290), (F32, 70000)])
def test_sampling_of_long_rows_at_every_alignment(dev, dtype, V):
    g = torch.Generator().manual_seed(V)
    V = V - 1 if V == 1 << 20 else V
    wide = (torch.randn(4, V + 1, generator=g) * 2).to(dtype)
    z, u = wide.to(dev)[:, 1:], torch.rand(4, generator=g)
    for setting in (dict(), dict(top_k=1000, top_p=0.9), dict(top_p=0.3, temperature=0.4), dict(min_p=0.02)):
        want = [O.sample(F64(wide[i, 1:]), float(u[i]), **setting) for i in range(4)]
        got = sample_tokens(z, u.to(dev), **setting).tolist()
        assert all(a == b or near < V * 2.0 ** -42 for a, (b, near) in zip(got, want)), (got, want)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_sampling_of_odd_rows(dev, dtype):
    V = 20000
    g = torch.Generator().manual_seed(9)
    z = (torch.randn(12, V, generator=g) * 3)
    z[0, :] = 0.0
    z[1, 100:] = -0.0
    z[2] *= 1e-30            # all next to zero
    z[3] *= 1e4              # beyond the table
    z[4, 5:] = -1e30
    z[5] = z[5].round()
    z[6, 7] = 1e30
    z[7] = -70000.0
    z[8, ::2] = torch.finfo(torch.bfloat16).min
    z[9, :-1] = -torch.inf
    z[10] = z[10] * 1e-3 + 1e3
    z[11, 1::3] = torch.inf
    z = z.to(dtype)
    u = torch.rand(12, generator=g)
    for setting in (dict(), dict(temperature=1e-30), dict(temperature=1e30), dict(temperature=1e-3, top_p=0.9),
                    dict(top_k=15000), dict(top_k=15000, top_p=0.99), dict(top_p=1e-9), dict(min_p=1e-5, top_k=V - 1),
                    dict(temperature=100.0, top_k=40, top_p=0.6)):
        want = [O.sample(F64(z[i]), float(u[i]), **setting) for i in range(12)]
        got = sample_tokens(z.to(dev), u.to(dev), **setting).tolist()
        assert all(a == b or near < V * 2.0 ** -42 for a, (b, near) in zip(got, want)), (setting, got, want)
    each = sample_tokens(z.to(dev).view(3, 4, V), u.to(dev).view(3, 4), temperature=torch.full((3, 4), 0.5, device=dev),
                         top_k=torch.arange(12, device=dev).view(3, 4), top_p=torch.full((3, 4), 0.75, device=dev),
                         min_p=torch.zeros(3, 4, device=dev))
    want = [O.sample(F64(z[i]), float(u[i]), temperature=0.5, top_k=i, top_p=0.75)[0] for i in range(12)]
    assert each.shape == (3, 4) and each.flatten().tolist() == want
    beyond = torch.tensor([-0.5, 1.0, 7.0, float("nan")] * 3)
    assert ((sample_tokens(z.to(dev), beyond.to(dev), top_k=3) >= 0).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("off", [0, 1])
def test_sampling_of_the_longest_rows(dev, dtype, off):
    g = torch.Generator().manual_seed(off)
    V = 1 << 20
    wide = (torch.randn(3, V + 8, generator=g) * 2).to(dtype)
    z, u = wide.to(dev)[:, off:off + V], torch.rand(3, generator=g)
    for setting in (dict(), dict(top_k=1000, top_p=0.9)):
        want = [O.sample(F64(wide[i, off:off + V]), float(u[i]), **setting) for i in range(3)]
        got = sample_tokens(z, u.to(dev), **setting).tolist()
        assert all(a == b or near < V * 2.0 ** -42 for a, (b, near) in zip(got, want)), (got, want)
    z = torch.zeros(2, V, device=dev, dtype=dtype)  # all weights the largest
    assert sample_tokens(z, torch.tensor([0.25, 1 - 2.0 ** -24], device=dev)).tolist() == [V // 4, V - 1]


def test_other_head_sizes_of_the_same_rows_are_refused(dev):
    cache = random_cache(2, 2, 20, [50, 50], 16, dev, 9)
    with pytest.raises(ValueError, match="head size"):
        cached_attention(torch.zeros(2, 2, 1, 25, device=dev), cache, 40, tau(dev))
