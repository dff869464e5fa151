"""The gated feed-forward block where padding meets infinities."""
import math

import pytest
import torch

from paper_01_anti_decoy_pnfirtau_amd import ops  # noqa: F401  (loads the ops)
from paper_01_anti_decoy_pnfirtau_amd._lib import PNFX_ACT, PNFX_KEEP
from tests.helpers import seeded

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype,keep", [(BF16, "none"), (BF16, "full"), (BF16, "e4m3"), (F32, "none"), (F32, "full")])
@pytest.mark.parametrize("T,D,F", [(3, 1, 9), (3, 8, 33), (20, 16, 5), (70, 1, 9), (70, 8, 33), (300, 24, 70), (2600, 72, 4099)])
def test_infinite_rows_over_padded_columns(dev, T, D, F, dtype, keep, act):
    """The columns that F is rounded up by are zero whatever x holds: of an infinite row too, whose y is infinite by
    the formula (all weights are positive)."""
    print(f"[ffn inf {T} {D} {F} {dtype} {keep} {act}]", flush=True)
    x = seeded((T, D), 300, dtype, dev)
    w_in, w_down = (seeded(s, 301 + i, dtype, dev, 0.1).abs() + 0.01 for i, s in enumerate(((2 * F, D), (6, F))))
    bad = x.clone()
    bad[1] = math.inf
    ref = torch.ops.pnfx.gated_ffn(x, w_in, w_down, PNFX_ACT[act], PNFX_KEEP[keep])[0]
    y, gu, _ = torch.ops.pnfx.gated_ffn(bad, w_in, w_down, PNFX_ACT[act], PNFX_KEEP[keep])
    assert bool((y[1] == math.inf).all()), y[1]
    rest = torch.arange(T, device=dev) != 1
    assert torch.equal(y[rest], ref[rest])
    if keep != "none":
        assert not bool((gu[:, :, F:].float() != 0).any())  # (NaN is not zero)
