"""Cross entropy over the vocabulary where logits leave their ordinary range."""
import pytest
import torch

from paper_01_anti_decoy_pnfirtau_amd import ops  # noqa: F401  (loads the ops)
from paper_01_anti_decoy_pnfirtau_amd._lib import PNFX_REDUCE
from tests.test_gpu_xent import BF16, F32, make

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
