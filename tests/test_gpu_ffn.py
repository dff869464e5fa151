"""The gated feed-forward block (pnfx::gated_ffn and its backward) against its formulas in 64 bits.

The tolerances are elementwise bounds on the sum of the roundings that the kernels make, each at most half a
step: H = 2^-8 of the value where it is rounded to bf16, E = 2^-24 where it is an fp32 operation, (n + 2) E of the
absolute sum for an fp32 sum of n products.  |silu'| and |gelu'| are below 1.13, |silu''| and |gelu''| below 0.8.
"""
import math

import pytest
import torch

from paper_01_anti_decoy_pnfirtau_amd import gated_ffn, ops  # noqa: F401  (loads the ops)
from paper_01_anti_decoy_pnfirtau_amd._lib import PNFX_ACT, PNFX_KEEP
from tests.helpers import seeded

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
BF16, F32 = torch.bfloat16, torch.float32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def act64(v, act):
    """act(v) and act'(v)."""
    if act == "silu":
        p = torch.sigmoid(v)
        return v * p, p * (1 + v * (1 - p))
    p = torch.special.ndtr(v)
    return v * p, p + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)


def make(T, D, F, Do, dtype, dev, seed=0):
    return (seeded((T, D), seed, dtype, dev), seeded((2 * F, D), seed + 1, dtype, dev, D ** -0.5),
            seeded((Do, F), seed + 2, dtype, dev, F ** -0.5), seeded((T, Do), seed + 3, dtype, dev))


def forward64(x, w_in, w_down, act, H):
    """g, u, h and y in 64 bits with bounds on the kernel's errors of each (h and y rounded to the type)."""
    D, F = x.shape[1], w_down.shape[1]
    z, ez = x @ w_in.T, (D + 2) * E * (x.abs() @ w_in.abs().T)
    g, u, eg, eu = z[:, :F], z[:, F:], ez[:, :F], ez[:, F:]
    a, _ = act64(g, act)
    h = a * u
    # the activation's own arithmetic: some ten fp32 operations, of at most |g| where it cancels
    eh = 1.13 * eg * u.abs() + (a.abs() + 1.13 * eg) * eu + 16 * E * g.abs() * u.abs()
    eh = eh + H * (h.abs() + eh)
    y = h @ w_down.T
    ey = eh @ w_down.abs().T + (F + 2) * E * ((h.abs() + eh) @ w_down.abs().T)
    return (g, eg), (u, eu), (h, eh), (y, ey + H * (y.abs() + ey))


def backward64(dy, x, w_in, w_down, act, g, eg, u, eu, H):
    """The gradients at g and u, of which the kernel has values at most eg and eu off, and their bounds."""
    T, D = x.shape
    Do, F = w_down.shape
    a, s = act64(g, act)
    ea, es = 1.13 * eg + 16 * E * g.abs(), 0.8 * eg + 16 * E * (1 + g.abs())
    dh, edh = dy @ w_down, (Do + 2) * E * (dy.abs() @ w_down.abs())
    prod = lambda p, ep, q, eq: (p * q, p.abs() * eq + ep * q.abs() + ep * eq + E * (p * q).abs())  # noqa: E731
    rnd = lambda v, e: (v, e + H * (v.abs() + e))  # noqa: E731
    dg, edg = rnd(*prod(*prod(dh, edh, u, eu), s, es))
    du, edu = rnd(*prod(dh, edh, a, ea))
    h, eh = rnd(*prod(a, ea, u, eu))
    d, ed = torch.cat([dg, du], 1), torch.cat([edg, edu], 1)

    def mm(p, ep, q, n):  # p with error, q exact
        v, mass = p @ q, (p.abs() + ep) @ q.abs()
        return rnd(v, ep @ q.abs() + (n + 66) * E * mass)  # 64 more for the sum of splits

    return (mm(d, ed, w_in, 2 * F), mm(d.T, ed.T, x, T),
            tuple(t.T for t in mm(h.T, eh.T, dy, T)))


def close(got, want, what):
    (v, e), got = want, got.double()
    assert got.shape == v.shape, (what, got.shape, v.shape)
    over = (got - v).abs() - e
    assert bool((over <= 0).all()), (what, float(over.max()), float((got - v).norm() / v.norm()))
    # the bounds add up absolute values: what is systematically wrong shows in the norm
    assert float((got - v).norm()) <= 4 * float(e.max() / v.abs().max().clamp(min=1e-30)) * float(v.norm()) + 1e-30, what


CASES = [
    # T, D, F, Do
    (1, 8, 8, 8), (1, 1, 1, 1), (3, 5, 7, 9), (16, 64, 64, 64), (17, 72, 40, 33), (64, 200, 96, 200),
    (65, 64, 128, 64), (100, 250, 66, 130), (129, 40, 300, 24), (257, 136, 129, 264), (300, 33, 31, 65),
    (520, 64, 520, 512),
]


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T,D,F,Do", CASES)
def test_forward_and_gradients(dev, T, D, F, Do, dtype, act):
    print(f"[ffn {T} {D} {F} {Do} {dtype} {act}]", flush=True)
    x, w_in, w_down, dy = make(T, D, F, Do, dtype, dev)
    H = half_step(dtype)
    x64, wi64, wd64, dy64 = (t.double() for t in (x, w_in, w_down, dy))
    (g, eg), (u, eu), _, y64 = forward64(x64, wi64, wd64, act, H)
    close(gated_ffn(x, w_in, w_down, act), y64, "y without gradient")
    leaves = [t.clone().requires_grad_() for t in (x, w_in, w_down)]
    y = gated_ffn(*leaves, activation=act)
    close(y.detach(), y64, "y")
    got = torch.autograd.grad(y, leaves, dy)
    if dtype == BF16:
        # kept in half precision: 2^-11 of the value, or half of its smallest step, 2^-24, times the block's
        # power of two, of which the largest value is at least 2^14
        tops = [torch.nn.functional.pad(t.abs(), (0, -F % 32)).view(T, -1, 32).amax(2).repeat_interleave(32, 1)[:, :F]
                for t in (g, u)]
        eg, eu = (e + 2.0 ** -11 * (t.abs() + e) + 2.0 ** -39 * m for t, e, m in zip((g, u), (eg, eu), tops))
    for name, a, want in zip(("dx", "dw_in", "dw_down"), got,
                             backward64(dy64, x64, wi64, wd64, act, g, eg, u, eu, H)):
        assert a.dtype == dtype
        close(a, want, name)


@pytest.mark.parametrize("dtype,T,D,F,Do", [
    (BF16, 2100, 520, 2060, 520),   # 256-tiles forward, k shared by two groups of waves backward
    (BF16, 4100, 2056, 4104, 2056),  # 256-tiles throughout
    (F32, 700, 300, 500, 300),      # splits of k, summed by another kernel
])
def test_larger_tiles_and_splits(dev, dtype, T, D, F, Do):
    test_forward_and_gradients(dev, T, D, F, Do, dtype, "silu")


def e4m3(b):
    return b.view(torch.float8_e4m3fn).double()


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("T,D,F,Do", [(1, 8, 8, 8), (3, 5, 7, 9), (65, 64, 128, 64), (100, 250, 66, 130),
                                      (300, 33, 31, 65), (520, 64, 520, 512)])
def test_eight_bit_checkpoint(dev, T, D, F, Do, act):
    """The bytes are within half an e4m3 step of g and u, their scale the smallest that holds the block,
    and the gradients are the formula's at exactly the values the bytes stand for."""
    print(f"[ffn e4m3 {T} {D} {F} {Do} {act}]", flush=True)
    x, w_in, w_down, dy = make(T, D, F, Do, BF16, dev, 10)
    x[0] *= 50.0  # blocks of another magnitude
    H = half_step(BF16)
    x64, wi64, wd64, dy64 = (t.double() for t in (x, w_in, w_down, dy))
    (g, eg), (u, eu), _, y64 = forward64(x64, wi64, wd64, act, H)
    y, gu, scales = torch.ops.pnfx.gated_ffn(x, w_in, w_down, PNFX_ACT[act], PNFX_KEEP["e4m3"])
    close(y, y64, "y")
    Fp, nb = (F + 7) // 8 * 8, (F + 31) // 32
    assert gu.shape == (T, 2, Fp) and scales.shape == (T, 2, nb)
    s = torch.ldexp(torch.ones((), dtype=torch.float64, device=dev), scales.int() - 127)
    s = s.repeat_interleave(32, 2)[:, :, :Fp]
    kept = e4m3(gu) * s
    assert not bool(kept[:, :, F:].any())
    kept, s = kept[:, :, :F], s[:, :, :F]
    v, ev = torch.stack([g, u], 1), torch.stack([eg, eu], 1)
    step = torch.maximum(v.abs() * 2.0 ** -4, s * 2.0 ** -10)
    assert bool(((kept - v).abs() <= step + 2 * ev).all())
    pad = torch.nn.functional.pad(v.abs() - ev, (0, nb * 32 - F)).view(T, 2, nb, 32).amax(3)
    top = torch.nn.functional.pad(v.abs() + ev, (0, nb * 32 - F)).view(T, 2, nb, 32).amax(3)
    sb = s[:, :, ::32]
    assert bool((pad <= 448 * sb).all()) and bool((top > 224 * sb).all())
    leaves = [t.clone().requires_grad_() for t in (x, w_in, w_down)]
    yt = gated_ffn(*leaves, activation=act, checkpoint="e4m3")
    assert torch.equal(yt.detach(), y)
    zero = torch.zeros_like(g)
    want = backward64(dy64, x64, wi64, wd64, act, kept[:, 0], zero, kept[:, 1], zero, H)
    for name, a, w in zip(("dx", "dw_in", "dw_down"), torch.autograd.grad(yt, leaves, dy), want):
        close(a, w, name)


def test_gradients_against_differences(dev):
    """Central differences of the fp32 forward along random directions."""
    x, w_in, w_down, dy = make(130, 48, 72, 40, F32, dev, 20)
    leaves = [t.clone().requires_grad_() for t in (x, w_in, w_down)]
    grads = torch.autograd.grad(gated_ffn(*leaves), leaves, dy)
    eps = 2.0 ** -7
    for i, g in enumerate(grads):
        v = seeded(g.shape, 30 + i, F32, dev)
        v /= v.norm()
        hi, lo = ([t + s * eps * v if j == i else t for j, t in enumerate((x, w_in, w_down))]
                  for s in (1.0, -1.0))
        f = lambda t: (gated_ffn(*t).double() * dy.double()).sum()  # noqa: E731
        num, ana = float((f(hi) - f(lo)) / (2 * eps)), float((g.double() * v.double()).sum())
        # third derivatives times eps^2 / 6 and the forward's roundings over eps
        assert abs(num - ana) <= 2e-3 * float(g.double().norm()), (i, num, ana)


def test_strides_views_and_leading_dims(dev):
    """Row strides, offset bases, several leading dimensions, a broadcast row and a transposed weight give the
    results of their contiguous copies, bit for bit; gradients come in the operands' shapes."""
    D, F = 64, 96
    wide = seeded((2, 40, D + 24), 40, BF16, dev)
    x = wide[:, :, 8:8 + D]
    w_in, w_down = seeded((D, 2 * F), 41, BF16, dev, 0.1).t(), seeded((D, F + 3), 42, BF16, dev, 0.1)[:, 3:]
    leaves = [t.detach().requires_grad_() for t in (x, w_in, w_down)]
    flat = [t.detach().contiguous().requires_grad_() for t in leaves]
    y, y2 = gated_ffn(*leaves), gated_ffn(*flat)
    assert y.shape == (2, 40, D) and torch.equal(y, y2)
    dy = seeded((2, 40, 1), 43, BF16, dev).expand(2, 40, D)
    for a, b, t in zip(torch.autograd.grad(y, leaves, dy), torch.autograd.grad(y2, flat, dy.contiguous()), leaves):
        assert a.shape == t.shape and torch.equal(a, b)
    odd = wide[:, :, 1:1 + D]  # two bytes off a 16-byte boundary
    assert torch.equal(gated_ffn(odd, w_in, w_down), gated_ffn(odd.contiguous(), w_in, w_down))
    row = seeded((1, D), 44, BF16, dev).expand(70, D)
    assert torch.equal(gated_ffn(row, w_in, w_down), gated_ffn(row.contiguous(), w_in, w_down))
    one = seeded((D,), 45, BF16, dev)
    assert torch.equal(gated_ffn(one, w_in, w_down), gated_ffn(one[None], w_in, w_down)[0])


def test_empty_and_partial_gradients(dev):
    x, w_in, w_down, _ = make(70, 64, 32, 64, BF16, dev, 50)
    none = x[:0].requires_grad_()
    w = w_in.clone().requires_grad_()
    y = gated_ffn(none, w, w_down)
    assert y.shape == (0, 64)
    gx, gw = torch.autograd.grad(y.sum(), (none, w))
    assert gx.shape == (0, 64) and not bool(gw.any())
    full = [t.clone().requires_grad_() for t in (x, w_in, w_down)]
    ref = torch.autograd.grad(gated_ffn(*full).sum(), full)
    for i in range(3):
        part = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, w_in, w_down))]
        assert torch.equal(torch.autograd.grad(gated_ffn(*part).sum(), part[i])[0], ref[i])


@pytest.mark.parametrize("keep", ["full", "e4m3"])
def test_not_finite_rows_stay_in_their_rows(dev, keep):
    """A row of x that holds an infinity or a NaN leaves the other rows of y and dx as they are."""
    x, w_in, w_down, dy = make(200, 72, 50, 72, BF16, dev, 60)
    bad = x.clone()
    bad[17, 3], bad[190, 71] = float("inf"), float("nan")
    outs = []
    for t in (x, bad):
        t = t.clone().requires_grad_()
        y = gated_ffn(t, w_in, w_down, checkpoint=keep)
        outs.append((y.detach(), torch.autograd.grad(y, t, dy)[0]))
    rest = [i for i in range(200) if i not in (17, 190)]
    for a, b in zip(*outs):
        assert torch.equal(a[rest], b[rest])
    assert bool(outs[1][0][17].isnan().any()) and bool(outs[1][0][190].isnan().all())


def test_large_values_follow_the_formula(dev):
    """Gates far out on both sides: act(g) is g or 0 there, and its slope 1 or 0."""
    x = torch.tensor([[300.0], [-300.0], [0.0], [-0.0]], device=dev)
    w_in, w_down = torch.ones(2, 1, device=dev), torch.ones(1, 1, device=dev)
    for act in ("silu", "gelu"):
        t = x.clone().requires_grad_()
        y = gated_ffn(t, w_in, w_down, act)
        assert y.flatten().tolist() == [90000.0, 0.0, 0.0, 0.0]
        # d (act(x) x) / dx = act'(x) x + act(x)
        assert torch.autograd.grad(y.sum(), t)[0].flatten().tolist() == [600.0, 0.0, 0.0, 0.0]


def test_repeatable_on_a_side_stream_and_in_a_graph(dev):
    """The same bits on another stream, from two streams at once, and from replays of a captured training
    call with new inputs, eager work between them."""
    x, w_in, w_down, dy = make(700, 128, 192, 128, BF16, dev, 70)
    leaves = [t.clone().requires_grad_() for t in (x, w_in, w_down)]

    def call():
        y = gated_ffn(*leaves, checkpoint="e4m3")
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    ref = call()
    side = [torch.cuda.Stream() for _ in range(2)]
    got = []
    torch.cuda.synchronize()
    for s in side:
        with torch.cuda.stream(s):
            got.append(call())
    torch.cuda.synchronize()
    for outs in got:
        assert all(torch.equal(a, b) for a, b in zip(outs, ref))
    s = side[0]
    with torch.cuda.stream(s):
        call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = call()
    for i in range(3):
        with torch.no_grad():
            leaves[0].copy_(seeded(x.shape, 80 + i, BF16, dev))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(static, call()):
            assert torch.equal(a, b)
        torch.cuda.synchronize()


def test_refusals(dev):
    x, w_in, w_down, dy = make(4, 16, 8, 16, BF16, dev)
    with pytest.raises(TypeError):
        gated_ffn(x, w_in.float(), w_down)
    with pytest.raises(TypeError):
        gated_ffn(x.half(), w_in.half(), w_down.half())
    for bad in ((x[:, :8], w_in, w_down), (x, w_in[:15], w_down), (x, w_in, w_down[:, :7]),
                (x, w_in, w_down[0])):
        with pytest.raises(ValueError):
            gated_ffn(*bad)
    with pytest.raises(ValueError):
        gated_ffn(x, w_in, w_down.cpu())
    with pytest.raises(ValueError, match="8-bit"):
        gated_ffn(x.float().requires_grad_(), w_in.float(), w_down.float(), checkpoint="e4m3")
    y, gu, scales = torch.ops.pnfx.gated_ffn(x, w_in, w_down, 0, 1)
    bwd = torch.ops.pnfx.gated_ffn_bwd
    mask = [True, True, True]
    with pytest.raises(ValueError):
        bwd(dy, x, w_in, w_down, gu[:2], scales, 0, 1, mask)
    with pytest.raises(TypeError):
        bwd(dy, x, w_in, w_down, gu, scales, 0, 2, mask)
    with pytest.raises(ValueError):
        bwd(dy[:3], x, w_in, w_down, gu, scales, 0, 1, mask)
    t = x.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(gated_ffn(t, w_in, w_down).sum(), t, create_graph=True)
