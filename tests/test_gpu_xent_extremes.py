"""Cross entropy over the vocabulary where logits leave their ordinary range: NaN weights, and tokens masked with the
type's lowest value.

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
