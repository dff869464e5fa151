"""Cross entropy over the vocabulary where logits leave their ordinary range: NaN weights, tokens masked with the type's
lowest value, rows of nothing else, and offsets that all of a row's logits share.

E = 2^-24 of one fp32 operation, H half a step of the operands' type, as in test_gpu_xent.py.
"""
import math

import pytest
import torch

from paper_01_anti_decoy_pnfirtau_amd import linear_cross_entropy
from paper_01_anti_decoy_pnfirtau_amd._lib import PNFX_REDUCE
from tests.helpers import seeded
from tests.test_gpu_xent import BF16, E, F32, close, make, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,D,V", [(BF16, 24, 8192), (BF16, 96, 8192), (BF16, 136, 8192), (BF16, 256, 8192),
                                       (BF16, 320, 8192), (BF16, 520, 16384), (F32, 24, 8192)])
def test_nan_weights_make_every_loss_nan(dev, dtype, D, V):
    """A block of weight rows gone NaN, in front of several tiles of finite ones of the same workgroup."""
    print(f"[xent nan block {dtype} D={D} V={V}]", flush=True)
    T = 16384  # 128 x 64 tiles of 128, or 64 x 64 of 256: two or more for a workgroup
    x, w, target = make(T, D, V, dtype, dev, 0.1, 100)
    w[:128] = float("nan")
    target = torch.where(target >= 0, target.clamp(min=128), target)
    loss, _, lse = torch.ops.pnfx.linear_xent(x, w, target, -100, PNFX_REDUCE["none"])
    kept = target != -100
    assert bool(loss[kept].isnan().all()) and bool(lse[kept].isnan().all())
    assert not bool(loss[~kept].any())


# tiles of 128 tokens with the rows' fragments in registers (D <= 256), without, of 256, and in fp32; several for a workgroup
MASKED = [(BF16, 300, 8, 2000), (BF16, 300, 64, 2000), (BF16, 300, 96, 2000), (BF16, 300, 200, 2000),
          (BF16, 300, 256, 2000), (BF16, 300, 320, 2000), (BF16, 2600, 520, 6000), (F32, 300, 40, 2000),
          (BF16, 16384, 24, 8192), (BF16, 16384, 256, 8192), (F32, 16384, 24, 8192)]


@pytest.mark.parametrize("mask", ["lowest", "1e30", "1e10"])
@pytest.mark.parametrize("dtype,T,D,V", MASKED)
def test_masked_tokens_change_nothing(dev, dtype, T, D, V, mask):
    """Tokens whose logits are the type's lowest value (or far below the others): loss and gradients are those of the
    vocabulary without them, whole lanes, waves and tiles of masked tokens among them."""
    print(f"[xent masked {dtype} {T} {D} {V} {mask}]", flush=True)
    x, w, target = make(T, D, V, dtype, dev, 0.1, 110)
    x[:, 0] = 1.0
    w[:, 0] = 0.0
    out = torch.zeros(V, dtype=torch.bool, device=dev)
    out[:300], out[700:720], out[V - 333:] = True, True, True
    low = torch.finfo(dtype).min if mask == "lowest" else -float(mask)
    w[out] = 0.0
    w[out, 0] = low
    place = torch.cumsum(~out, 0) - 1
    inside = (~out).nonzero()[:, 0]
    target = torch.where(target >= 0, inside[target.clamp(min=0) % len(inside)], target)
    H = torch.finfo(dtype).eps / 2
    s = torch.ones(T, dtype=torch.float64, device=dev)
    (losses, el), dx, (dw, edw) = reference(x, w[inside], torch.where(target >= 0, place[target.clamp(min=0)], target), H, s)
    leaves = [t.clone().requires_grad_() for t in (x, w)]
    loss = linear_cross_entropy(*leaves, target, reduction="none")
    close(loss.detach(), (losses, el), "loss of each row")
    total = linear_cross_entropy(*leaves, target, reduction="sum")
    close(total.detach(), (losses.sum(), el.sum() + 2 * E * losses.sum()), "loss")
    got = torch.autograd.grad(total, leaves)
    close(got[0], dx, "dx")
    close(got[1][inside], (dw, edw), "dw")
    assert not bool(got[1][out].any())


@pytest.mark.parametrize("dtype,D", [(BF16, 8), (BF16, 72), (BF16, 256), (BF16, 320), (F32, 8)])
def test_minus_infinity_masks_tokens(dev, dtype, D):
    x, w, target = make(300, D, 2000, dtype, dev, 0.1, 120)
    x[:, 0], w[:, 0] = 1.0, 0.0
    w[:400], w[1800:] = 0.0, 0.0
    w[:400, 0], w[1800:, 0] = -math.inf, -math.inf
    target = torch.where(target >= 0, 400 + target % 1400, target)
    losses, el = reference(x, w[400:1800], torch.where(target >= 0, target - 400, target), 0.0)[0]
    close(linear_cross_entropy(x, w, target, reduction="none"), (losses, el), "loss")


@pytest.mark.parametrize("dtype,D", [(BF16, 8), (BF16, 72), (BF16, 256), (BF16, 320), (F32, 8)])
def test_rows_whose_every_token_is_masked(dev, dtype, D):
    """Every logit the type's lowest value: a uniform softmax, log V, as log_softmax has it.  Every logit minus infinity: NaN."""
    T, V = 140, 2048
    x, w = torch.zeros(T, D, dtype=dtype, device=dev), torch.zeros(V, D, dtype=dtype, device=dev)
    x[:, 0] = 1.0
    x[:, 1] = 1.0
    w[:, 0] = torch.finfo(dtype).min
    target = (torch.arange(T, device=dev) * 5) % V
    leaves = [t.clone().requires_grad_() for t in (x, w)]
    loss = linear_cross_entropy(*leaves, target, reduction="none")
    assert bool(((loss.double() - math.log(V)).abs() <= 8 * E * math.log(V)).all())
    total = linear_cross_entropy(*leaves, target, reduction="sum")
    dw = torch.autograd.grad(total, leaves[1])[0]
    d = torch.full((T, V), 1 / V, dtype=torch.float64, device=dev)
    d[torch.arange(T, device=dev), target] -= 1
    # p: its exponent is as exact as the loss, and a few roundings of 11 at most; rounded to the type as it is, and so is the sum
    H = torch.finfo(dtype).eps / 2
    ed = (128 * E + H) * d.abs()
    want, e = d.T.sum(1), ed.T.sum(1) + (T + 66) * E * d.abs().T.sum(1)
    for c in (0, 1):
        close(dw[:, c], (want, e + H * (want.abs() + e)), "dw")
    w[:, 0] = -math.inf
    assert bool(linear_cross_entropy(x, w, target, reduction="none").isnan().all())


@pytest.mark.parametrize("reduction", ["sum", "none"])
@pytest.mark.parametrize("power", [8, 14, 20, 27, 30, 33, 60, 126])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("dtype,D", [(BF16, 8), (BF16, 72), (BF16, 256), (BF16, 320), (F32, 8)])
def test_shared_offsets_leave_softmax_alone(dev, dtype, D, sign, power, reduction):
    """Logits 2^power + k u with small whole k and a unit u that both types hold exactly: the logits are exact, and
    with them every difference that loss and gradients are made of, whatever the offset."""
    print(f"[xent offset {dtype} D={D} {sign} 2^{power} {reduction}]", flush=True)
    T, V = 150, 1300
    u = 2.0 ** max(0, power - 22)
    g = torch.Generator().manual_seed(power)
    a, b = torch.randint(0, 4, (T,), generator=g), torch.randint(-4, 5, (V,), generator=g)
    x, w = torch.zeros(T, D, dtype=dtype), torch.zeros(V, D, dtype=dtype)
    x[:, 0], x[:, 1] = 1.0, a.to(dtype)
    w[:, 0], w[:, 1] = sign * 2.0 ** power, (b * u).to(dtype)
    x, w, target = x.to(dev), w.to(dev), torch.randint(0, V, (T,), generator=g).to(dev)
    # the logits without their offset and their row's largest, which would take the digits of 64 bits, too
    k = (a[:, None] * b[None, :] * u).double().to(dev)
    k = k - k.amax(1, keepdim=True)
    lse = torch.logsumexp(k, 1, keepdim=True)
    want = (lse - k.gather(1, target[:, None]))[:, 0]
    leaves = [t.clone().requires_grad_() for t in (x, w)]
    rows = linear_cross_entropy(*leaves, target, reduction="none")
    # V sums of exponentials that are a few roundings off, and the difference of two exact logits, rounded
    el = 4 * E * want.abs() + (V + 64) * E
    close(rows.detach(), (want, el), "loss")
    loss = rows.sum() if reduction == "none" else linear_cross_entropy(*leaves, target, reduction="sum")
    dx, dw = torch.autograd.grad(loss, leaves)
    p = torch.exp(k - lse)
    # the exponent is rounded where it is up to ln V, and more where p is small; the reference of a row is as exact as its loss
    rel = 16 * E * ((k - lse).abs().clamp(max=88) + 8) + 4 * el[:, None]
    if power == 8:  # up to here the reference is the rounded log-sum-exp times log2 e: 2^-23 of it beside the exponent
        rel = rel + 2.0 ** power * 2 * E
    H = torch.finfo(dtype).eps / 2
    # (exponentials below fp32's normal range may come out as zero)
    d, ed = p.clone(), p * rel + 2.0 ** -126
    d.scatter_add_(1, target[:, None], -torch.ones_like(lse))
    ed.scatter_(1, target[:, None], (el + 4 * E)[:, None])
    ed = ed + H * (d.abs() + ed)
    x64, w64 = x.double(), w.double()
    # A row's statistics are fp32: of a loss and a log-sum-exp both far out, which are off by half a step, 2^-24 of
    # them, the softmax is known to a factor exp(2^-24 loss) only.  Where that is not near one (losses of 2^38 and more here)
    # tokens that tie at the top may get any share, up to 1 each, and with them dx of the row and every sum over rows.
    known = 4 * el < 0.125
    assert bool(known.all()) or power >= 60
    assert bool(known.any())
    want = d @ w64, (ed + (V + 66) * E * d.abs()) @ w64.abs()
    close(dx[known], (want[0][known], (want[1] + H * (want[0].abs() + want[1]))[known]), "dx")
    if bool(known.all()):
        v, e = d.T @ x64, (ed.T + (T + 66) * E * d.abs().T) @ x64.abs()
        close(dw, (v, e + H * (v.abs() + e)), "dw")
