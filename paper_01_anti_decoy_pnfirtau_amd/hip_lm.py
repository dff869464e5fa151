"""The language model's position-wise operators: the gated feed-forward block and the loss over the vocabulary.

================================  ==================================================================
``gated_ffn``                     ``(act(x Wg^T) * (x Wu^T)) Wd^T``
``linear_cross_entropy``          cross entropy of the logits ``x W^T``, which are never materialised
================================  ==================================================================

Neither has a counterpart in the reference, whose model takes torch's two-layer FFN and cross entropy
(experiments/exp4_wikitext2_lm.py:183-247, :334-348).  GPU tensors, bf16 or fp32, run the HIP kernels
(``pnfx::gated_ffn``, ``pnfx::linear_xent``); CPU tensors the same composition of torch operations.
Under autocast both compute in the autocast type, as ``nn.Linear`` does: the gradients of fp32 weights are
rounded to it, too.
"""
from __future__ import annotations

import functools

import torch
import torch.nn.functional as F

from . import _lib

ACTIVATIONS = ("silu", "gelu")
CHECKPOINTS = ("full", "e4m3")
REDUCTIONS = ("mean", "sum", "none")


@functools.cache
def _op(name: str):
    """The operator pnfx::name (importing ops loads the library, which CPU tensors do without)."""
    from . import ops  # noqa: F401

    return getattr(torch.ops.pnfx, name).default


def _one_of(what: str, value: str, choices: tuple[str, ...]) -> None:
    if value not in choices:
        raise ValueError(f"{what} {value!r}: one of {', '.join(choices)}")


def _autocast(*tensors: torch.Tensor) -> tuple[torch.Tensor, ...]:
    if not torch.is_autocast_enabled("cuda" if tensors[0].is_cuda else "cpu"):
        return tensors
    dtype = torch.get_autocast_dtype(tensors[0].device.type)
    return tuple(t.to(dtype) if t.is_floating_point() and t.dtype != torch.float64 else t
                 for t in tensors)


def gated_ffn(x: torch.Tensor, w_in: torch.Tensor, w_down: torch.Tensor, activation: str = "silu",
              checkpoint: str = "full") -> torch.Tensor:
    """The gated feed-forward block: ``(act(g) * u) @ w_down.T`` with ``g, u = (x @ w_in.T).chunk(2, -1)``.

    x [..., D], w_in [2 F, D] (the gate's rows, then the up projection's), w_down [D_out, F], all of one
    type; returns [..., D_out].  ``activation``: "silu", or "gelu" in its error-function form.

    Both projections, the activation and the product are one kernel; g, u and h = act(g) u are fp32 sums,
    and h is rounded to x's type for the second product.  Any sizes and row strides; operands whose
    inner size is not a multiple of 8, or that are not 16-byte aligned, are copied first.

    ``checkpoint``: how g and u are kept for the backward pass.  "full": in fp32 for fp32 operands, else in
    16 bits, half precision with a power of two for each block of 32 columns (2^-11 at most beside g and u, relative, or
    2^-39 of the block's largest).  "e4m3": in 8 bits with such scales, half the memory: 2^-4 at most beside g and
    u, relative, or 2^-10 of the block's scale; of bf16 operands, and a call that would have to keep fp32 ones
    so is refused (ValueError).  Where the kernels keep nothing, as no gradient is recorded or the tensors are on the
    CPU, both settings are taken and change nothing.  The gradients are those at the values that the kept ones
    stand for; y is the same.  The backward is bitwise repeatable; second derivatives and tangents (forward mode) are
    refused.
    """
    _one_of("activation", activation, ACTIVATIONS)
    _one_of("checkpoint", checkpoint, CHECKPOINTS)
    x, w_in, w_down = _autocast(x, w_in, w_down)
    if not x.is_cuda:
        g, u = F.linear(x, w_in).chunk(2, -1)
        return F.linear((F.silu(g) if activation == "silu" else F.gelu(g)) * u, w_down)
    keep = checkpoint if torch.is_grad_enabled() and (
        x.requires_grad or w_in.requires_grad or w_down.requires_grad) else "none"
    return _op("gated_ffn")(x, w_in, w_down, _lib.PNFX_ACT[activation], _lib.PNFX_KEEP[keep])[0]


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor,
                         ignore_index: int = -100, reduction: str = "mean") -> torch.Tensor:
    """``F.cross_entropy(x @ weight.T, target)`` without the logits: x [..., D], weight [V, D], target
    int64 [...].

    Returns fp32: one value ("mean" over the rows that are not ignored, "sum") or target's shape ("none").
    Rows whose target is ``ignore_index`` cost nothing, have loss and gradient 0 and, whatever they hold,
    reach no other result.  Another target outside 0 .. V - 1 makes its row's loss and gradients NaN (the
    host is never made to wait for a check; CPU tensors raise an IndexError).  Logits, maxima and sums are fp32;
    the gradient of the logits is rounded to x's type for the products with weight and x.  Before that its
    softmax is off by 2^-13 at most, relative (fp32 operands: 2^-18), beside the logits' own roundings, or by 2^-23 of a
    row's loss or log-sum-exp where the smaller of the two is larger than 1024 (32).  The memory beside the
    gradients is a piece of the vocabulary's logits, 256 MB or 2048 tokens' worth (none for bf16 rows of up to
    64 columns and one loss value), and fp32 sums of the gradients.  Bitwise repeatable; second derivatives and
    tangents (forward mode) are refused.

    In bf16 it is also the faster way (training 1.9 to 4.3 times F.linear and F.cross_entropy).  In fp32 the logits' second
    product mostly costs more than their memory traffic: 153 rows, D = 1952, 52097 tokens take 1670 us against 920, 4096 x
    512 x 33278 4430 against 4000, 333 x 1000 x 50257 1230 against 1390; there it is for logits that are not to be in
    memory.
    """
    _one_of("reduction", reduction, REDUCTIONS)
    x, weight = _autocast(x, weight)
    if not x.is_cuda:
        rows, to = x.reshape(-1, x.shape[-1]), target.reshape(-1)
        rows = torch.where((to != ignore_index).unsqueeze(1), rows, 0)  # what ignored rows hold reaches dW otherwise
        loss = F.cross_entropy(F.linear(rows, weight).float(), to, ignore_index=ignore_index, reduction=reduction)
        return loss.view(target.shape) if reduction == "none" else loss
    return _op("linear_xent")(x, weight, target, int(ignore_index), _lib.PNFX_REDUCE[reduction])[0]
