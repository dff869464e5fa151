"""The feed-forward block and the vocabulary cross entropy without a GPU: the CPU composition, the choices of the
language model, the operators' autograd and fake kernels, and what the C ABI refuses before any device call."""
import ctypes

import pytest
import torch
import torch.nn.functional as F

import paper_01_anti_decoy_pnfirtau_amd as P
from paper_01_anti_decoy_pnfirtau_amd import _lib
from paper_01_anti_decoy_pnfirtau_amd.wikilm import GatedFFN, WikiLM, WikiLMConfig, lm_loss, make_optimizer, train_step


def test_cpu_composition():
    g = torch.Generator().manual_seed(0)
    x, w_in, w_down = (torch.randn(s, generator=g) for s in ((2, 5, 8), (12, 8), (7, 6)))
    gate, up = F.linear(x, w_in).chunk(2, -1)
    for act, fn in (("silu", F.silu), ("gelu", F.gelu)):
        assert torch.equal(P.gated_ffn(x, w_in, w_down, act), F.linear(fn(gate) * up, w_down))
    w, target = torch.randn(11, 8, generator=g), torch.tensor([[0, 3, -100, 10, 1], [2, -100, 4, 4, 0]])
    for reduction in ("mean", "sum", "none"):
        got = P.linear_cross_entropy(x, w, target, reduction=reduction)
        ref = F.cross_entropy((x @ w.T).flatten(0, 1), target.flatten(), reduction=reduction)
        assert torch.allclose(got.flatten(), ref.flatten(), rtol=1e-6, atol=1e-6)
        assert got.shape == (target.shape if reduction == "none" else ())
    for call in (lambda: P.gated_ffn(x, w_in, w_down, "relu"), lambda: P.gated_ffn(x, w_in, w_down, checkpoint="int8"),
                 lambda: P.linear_cross_entropy(x, w, target, reduction="max")):
        with pytest.raises(ValueError, match="one of"):
            call()


@pytest.mark.parametrize("ffn", ["gelu", "swiglu", "geglu"])
def test_language_model_choices_on_cpu(ffn):
    """The fused loss is the loss of the materialised logits; a gated model trains; the default model's parameters
    are those it always had."""
    base = dict(d_model=32, n_heads=4, n_layers=2, d_ff=48, max_seq=32, dropout=0.0)
    x = torch.randint(0, 50, (2, 32), generator=torch.Generator().manual_seed(0))
    losses, grads = [], []
    for fused in (False, True):
        torch.manual_seed(1)
        m = WikiLM(50, WikiLMConfig(**base, ffn=ffn, fused_loss=fused), "pn_fir_tau")
        loss = lm_loss(m, x, amp=False)
        loss.backward()
        losses.append(loss.detach())
        grads.append([p.grad for p in m.parameters()])
        names = [n for n, _ in m.named_parameters()]
        assert ("blocks.0.ffn.gate_up.weight" in names) == (ffn != "gelu")
        assert ("blocks.0.ffn.0.weight" in names) == (ffn == "gelu")
        assert train_step(m, make_optimizer(m, m.cfg), x, amp=False).isfinite()
    assert torch.allclose(*losses, rtol=1e-6, atol=0)
    for a, b in zip(*grads):
        assert torch.allclose(a, b, rtol=1e-4, atol=1e-6)
    with pytest.raises(ValueError, match="Unknown ffn"):
        WikiLM(50, WikiLMConfig(**base, ffn="relu"), "pn_fir_tau")


def test_gated_ffn_module():
    m = GatedFFN(8, 12, "gelu", checkpoint="e4m3")
    assert m.gate_up.weight.shape == (24, 8) and m.down.weight.shape == (8, 12)
    x = torch.randn(3, 8)
    assert torch.equal(m(x), P.gated_ffn(x, m.gate_up.weight, m.down.weight, "gelu"))


def test_fake_kernels_give_the_outputs_layouts():
    from torch._subclasses.fake_tensor import FakeTensorMode

    from paper_01_anti_decoy_pnfirtau_amd import ops  # noqa: F401

    p = torch.ops.pnfx
    with FakeTensorMode(allow_non_fake_inputs=True):
        x = torch.empty(2, 5, 16, dtype=torch.bfloat16, device="cuda")
        w_in, w_down = x.new_empty(74, 16), x.new_empty(9, 37)
        for keep, shape, dtype, scales in ((0, (0,), None, (0,)), (1, (10, 2, 40), torch.float16, (10, 2, 2)),
                                           (2, (10, 2, 40), torch.uint8, (10, 2, 2))):
            y, gu, sc = p.gated_ffn(x, w_in, w_down, 0, keep)
            assert y.shape == (2, 5, 9) and gu.shape == shape and sc.shape == scales and sc.dtype == torch.uint8
            assert dtype is None or gu.dtype == dtype
        f = p.gated_ffn(x.float(), w_in.float(), w_down.float(), 1, 1)
        assert f[1].dtype == torch.float32 and f[2].shape == (0,)
        d = p.gated_ffn_bwd(y, x, w_in, w_down, gu, sc, 0, 2, [True, False, True])
        assert [t.shape for t in d] == [x.shape, (0,), w_down.shape]
        w, t = x.new_empty(33, 16), torch.empty(2, 5, dtype=torch.long, device="cuda")
        for reduction, shape in ((0, (2, 5)), (1, ()), (2, ())):
            loss, rows, lse = p.linear_xent(x, w, t, -100, reduction)
            assert loss.shape == shape and loss.dtype == torch.float32 and rows.shape == lse.shape == (10,)
        d = p.linear_xent_bwd(loss, x, w, t, rows, lse, -100, 2, [False, True])
        assert [t.shape for t in d] == [(0,), w.shape]


def test_c_abi_refuses_bad_arguments_on_the_host():
    """Before any device call: the pointers are never followed."""
    lib = _lib.lib()
    p, odd, big = ctypes.c_void_p(256), ctypes.c_void_p(264), 1 << 40

    def fwd(T=4, D=16, Fd=8, Do=16, x=p, rs=(16, 16, 8), y=p, gu=p, sc=p, act=0, keep=1, dtype=1, ws=p, wsb=big):
        return lib.pnfx_ffn_fwd(x, rs[0], p, rs[1], p, rs[2], y, gu, sc, T, D, Fd, Do, act, keep, dtype, ws, wsb, None)

    def bwd(T=4, D=16, Fd=8, Do=16, gu=p, sc=p, dx=p, act=0, keep=1, dtype=1, ws=p, wsb=big, rs=16):
        return lib.pnfx_ffn_bwd(p, rs, p, 16, p, 16, p, 8, gu, sc, dx, p, p, T, D, Fd, Do, act, keep, dtype, ws, wsb, None)

    for kw in (dict(x=None), dict(y=None), dict(T=0), dict(D=0), dict(Fd=1 << 19), dict(T=1 << 30), dict(rs=(15, 16, 8)),
               dict(rs=(16, 16, 7)), dict(act=2), dict(keep=3), dict(keep=2, dtype=0), dict(dtype=2), dict(gu=None),
               dict(sc=None), dict(ws=None), dict(wsb=16), dict(y=odd), dict(ws=odd)):
        assert fwd(**kw) == -1, kw
    for kw in (dict(gu=None), dict(sc=None), dict(keep=0), dict(keep=2, dtype=0), dict(dx=odd), dict(gu=odd), dict(T=0),
               dict(ws=None), dict(wsb=16), dict(rs=15), dict(act=-1)):
        assert bwd(**kw) == -1, kw
    assert b"row strides" in lib.pnfx_last_error() or lib.pnfx_last_error()

    def xent(T=4, D=16, V=20, x=p, target=p, loss=p, rs=16, reduction=2, dtype=1, ws=p, wsb=big):
        return lib.pnfx_xent_fwd(x, rs, p, 16, target, -100, loss, p, p, T, D, V, reduction, dtype, ws, wsb, None)

    def xent_b(T=4, D=16, V=20, dloss=p, dx=p, rs=16, reduction=2, dtype=1, ws=p, wsb=big):
        return lib.pnfx_xent_bwd(dloss, p, rs, p, 16, p, -100, p, p, dx, p, T, D, V, reduction, dtype, ws, wsb, None)

    for kw in (dict(x=None), dict(target=None), dict(loss=None), dict(T=0), dict(V=0), dict(V=1 << 25), dict(T=1 << 25),
               dict(D=1 << 19), dict(rs=8), dict(reduction=3), dict(dtype=7), dict(ws=None), dict(wsb=64), dict(ws=odd)):
        assert xent(**kw) == -1, kw
    for kw in (dict(dloss=None), dict(dx=odd), dict(rs=8), dict(reduction=-1), dict(wsb=64), dict(D=0)):
        assert xent_b(**kw) == -1, kw
    assert lib.pnfx_ffn_fwd_workspace_size(0, 8, 8, 8, 0, 0, 1) == 0
    assert lib.pnfx_xent_bwd_workspace_size(4, 8, 0, 2, 0, 1) == 0


@pytest.mark.parametrize("T,D,V,dtype", [(16384, 256, 33278, 1), (1, 8, 2, 1), (200000, 64, 32000, 1), (2048, 256, 8191, 0)])
def test_cross_entropy_workspace_is_bounded_by_a_piece(T, D, V, dtype):
    """The backward's workspace holds 256 MB of logits' gradients at most (or 2048 tokens' worth), never all of them,
    beside x-sized buffers and the fp32 sums of the two gradients."""
    es = 2 if dtype else 4
    got = _lib.lib().pnfx_xent_bwd_workspace_size(T, D, V, 2, 0, dtype)
    piece = min(max(256 << 20, 2048 * T * es), T * (V + 7) * es) + 256 * T * es
    assert got <= piece + 2 * T * (D + 8) * es + 40 * T + 80 * T * D * 4 + 80 * (V + 256) * D * 4 + 65536


def test_operators_refuse_cpu_tensors_and_second_derivatives():
    from paper_01_anti_decoy_pnfirtau_amd import ops  # noqa: F401

    x, w = torch.randn(3, 8), torch.randn(16, 8)
    with pytest.raises(Exception):
        torch.ops.pnfx.gated_ffn(x, w, torch.randn(8, 8), 0, 0)
    with pytest.raises(Exception):
        torch.ops.pnfx.linear_xent(x, w, torch.zeros(3, dtype=torch.long), -100, 0)
