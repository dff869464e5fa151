"""The language model's operators where a workgroup has more than one tile, stage or piece to go through: loops that
small sizes leave after their first pass.  References and bounds are those of test_gpu_ffn.py and test_gpu_xent.py.
"""
import pytest
import torch

from paper_01_anti_decoy_pnfirtau_amd import _lib, gated_ffn, linear_cross_entropy
from tests.helpers import seeded
from tests.test_gpu_ffn import close as ffn_close
from tests.test_gpu_ffn import forward64, half_step, test_eight_bit_checkpoint as eight_bit
from tests.test_gpu_ffn import make as ffn_make
from tests.test_gpu_xent import BF16, E, F32, close, make, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T", [1, 16, 20, 40, 48, 64])
@pytest.mark.parametrize("D,F,Do", [(1100, 4200, 1100), (1096, 2311, 1333), (4099, 700, 260)])
def test_few_rows_over_a_long_k(dev, T, D, F, Do, dtype, act):
    """Inference of up to 64 rows whose waves go round their ring of stages several times (a piece of k is 128 bytes,
    four or eight waves take turns, and two to four pieces of each are on their way)."""
    print(f"[ffn rows {T} {D} {F} {Do} {dtype} {act}]", flush=True)
    x, w_in, w_down, _ = ffn_make(T, D, F, Do, dtype, dev, 200)
    *_, y = forward64(*(t.double() for t in (x, w_in, w_down)), act, half_step(dtype))
    ffn_close(gated_ffn(x, w_in, w_down, act), y, "y")


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("T,D,F,Do", [(4100, 2056, 4104, 2056), (2100, 520, 2060, 520)])
def test_eight_bits_in_large_tiles(dev, T, D, F, Do, act):
    """256-tiles forward and backward, and tiles whose k two groups of waves share, with the projections kept in 8 bits."""
    eight_bit(dev, T, D, F, Do, act)


def tiles_of_a_workgroup(T, D, V, dtype, tile):
    """The forward's vocabulary tiles for each workgroup, from the workspace that its statistics take."""
    es, code = (2, _lib.PNFX_BF16) if dtype == BF16 else (4, _lib.PNFX_F32)
    total = _lib.lib().pnfx_xent_fwd_workspace_size(T, D, V, 0, code)
    rest = T * D * es + 3 * T * 4  # the kept rows and three words of each
    splits = round((total - rest) / (T * 8 * 4))  # four waves' maximum and sum
    return -(-V // tile) / splits


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("dtype,T,D,V,tile", [
    # rows' fragments in registers, one to four steps of k: four tiles of a workgroup backward too, so that stores of
    # several are on their way (of one step only for a loss per row); two to four pieces of the vocabulary
    (BF16, 16384, 64, 24576, 128), (BF16, 16384, 128, 32768, 128), (BF16, 16384, 192, 24576, 128),
    (BF16, 16384, 256, 32768, 128),
    # the loop over k: five steps, a last tile and a last piece that are not whole
    (BF16, 16384, 320, 20001, 128), (F32, 16384, 96, 16388, 128),
    # 256-tiles, two of a workgroup backward too
    (BF16, 131072, 512, 4096, 256),
])
def test_many_tiles_and_pieces(dev, dtype, T, D, V, tile, reduction):
    """The rows' maxima grow by 12 from tile to tile, so that sums are rescaled, and fall back every fourth."""
    print(f"[xent tiles {dtype} {T} {D} {V} {reduction}]", flush=True)
    assert tiles_of_a_workgroup(T, D, V, dtype, tile) >= 3.9
    x, w, target = make(T, D, V, dtype, dev, 0.05, 210)
    x[:, 0] = 1.0
    w[:, 0] = (torch.arange(V, device=dev) // tile % 4 * 12).to(dtype)
    H = torch.finfo(dtype).eps / 2
    kept = int((target != -100).sum())
    dloss = seeded((T,) if reduction == "none" else (), 5, F32, dev)
    s = dloss.double().expand(T) / (kept if reduction == "mean" else 1)
    (losses, el), *grads = reference(x, w, target, H, s, per_row=reduction == "none")
    if reduction == "mean":
        losses, el = losses.sum() / kept, el.sum() / kept + 2 * E * losses.sum() / kept
    leaves = [t.clone().requires_grad_() for t in (x, w)]
    loss = linear_cross_entropy(*leaves, target, reduction=reduction)
    close(loss.detach(), (losses, el), "loss")
    for name, a, want in zip(("dx", "dw"), torch.autograd.grad(loss, leaves, dloss), grads):
        close(a, want, name)
