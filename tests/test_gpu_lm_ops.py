"""The feed-forward block and the vocabulary cross entropy together, as the language model trains with them."""
import pytest
import torch
import torch.nn.functional as F

from paper_01_anti_decoy_pnfirtau_amd import gated_ffn, linear_cross_entropy, ops  # noqa: F401
from paper_01_anti_decoy_pnfirtau_amd.wikilm import (GATED_FFN, GraphedStep, WikiLM, WikiLMConfig, lm_loss,
                                                      make_optimizer, train_step)
from tests.helpers import seeded

pytestmark = pytest.mark.gpu

VOCAB = 300
BASE = dict(d_model=64, n_heads=4, n_layers=2, d_ff=96, max_seq=128, dropout=0.0)


def model(dev, seed=0, **choices):
    torch.manual_seed(seed)
    return WikiLM(VOCAB, WikiLMConfig(**BASE, **choices), "pn_fir_tau_flash").to(dev)


def batches(dev, n, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, VOCAB, (4, 128), generator=g).to(dev) for _ in range(n)]


def plain_loss(m, x, act):
    """lm_loss with the FFN and the loss as torch has them."""

    class Plain(torch.nn.Module):
        def __init__(self, f):
            super().__init__()
            self.f = f

        def forward(self, h):
            g, u = F.linear(h, self.f.gate_up.weight).chunk(2, -1)
            return F.linear((F.silu(g) if act == "silu" else F.gelu(g)) * u, self.f.down.weight)

    kept = [b.ffn for b in m.blocks]
    for b in m.blocks:
        b.ffn = Plain(b.ffn)
    try:
        logits = m(x)
        return F.cross_entropy(logits[:, :-1].flatten(0, 1), x[:, 1:].flatten())
    finally:
        for b, f in zip(m.blocks, kept):
            b.ffn = f


@pytest.mark.parametrize("ffn", ["swiglu", "geglu"])
def test_model_gradients_match_torch_fp32(dev, ffn):
    """Every parameter's gradient of the first step in fp32, within 1e-4 of its scale of the model with torch's
    FFN and cross entropy (two layers of fp32 products in another order)."""
    print(f"[lm ops fp32 {ffn}]", flush=True)
    x = batches(dev, 1)[0]
    m = model(dev, ffn=ffn, fused_loss=True)
    loss = lm_loss(m, x, amp=False)
    names, params = zip(*m.named_parameters())
    got = torch.autograd.grad(loss, params)
    ref_loss = plain_loss(m, x, GATED_FFN[ffn])
    ref = torch.autograd.grad(ref_loss, params)
    assert abs(float(loss.detach()) - float(ref_loss.detach())) <= 1e-5 * abs(float(ref_loss.detach()))
    for n, a, b in zip(names, got, ref):
        assert float((a - b).abs().max()) <= 1e-4 * float(b.abs().max()), n


@pytest.mark.parametrize("keep,tol", [("full", 2e-2), ("e4m3", 6e-2)])
def test_model_gradients_under_autocast(dev, keep, tol):
    """Under bf16 autocast the gradients are near the fp32 model's: bf16 roundings of 2^-8 in some ten products
    one behind the other; e4m3 adds 2^-4 / sqrt 3 at most on g and u, of which each sum averages many."""
    x = batches(dev, 1)[0]
    m = model(dev, ffn="swiglu", ffn_checkpoint=keep, fused_loss=True)
    params = list(m.parameters())
    ref = torch.autograd.grad(plain_loss(m, x, "silu"), params)
    got = torch.autograd.grad(lm_loss(m, x, amp=True), params)
    a, b = (torch.cat([g.flatten() for g in gs]) for gs in (got, ref))
    assert float((a - b).norm()) <= tol * float(b.norm())


@pytest.mark.parametrize("amp,keep", [(True, "e4m3"), (True, "full"), (False, "full")])
def test_graphed_step_is_the_eager_step(dev, amp, keep):
    """The whole training step captured and replayed with new tokens: each replay's loss is the eager model's."""
    print(f"[lm ops graph amp={amp} {keep}]", flush=True)
    xs = batches(dev, 6, 3)
    make = lambda: model(dev, ffn="swiglu", ffn_checkpoint=keep, fused_loss=True)  # noqa: E731
    eager, graphed = make(), make()
    opt_e, opt_g = (make_optimizer(m, m.cfg, capturable=True) for m in (eager, graphed))
    static = xs[0].clone()
    g = GraphedStep(graphed, opt_g, static, amp=amp, warmup=2)
    for i, x in enumerate(xs[:4]):
        le = float(train_step(eager, opt_e, x, amp=amp))
        torch.cuda.synchronize()
        static.copy_(x)
        lg = float(g.replay())
        torch.cuda.synchronize()
        assert abs(le - lg) <= (1e-3 if amp else 1e-5) * abs(le), (i, le, lg)


def test_step_runs_with_dropout_and_checkpointing(dev):
    """Dropout, torch's activation checkpointing around the block, and saved tensors that come back elsewhere."""
    m = model(dev, ffn="geglu", fused_loss=True)
    m.drop.p = 0.1
    x = batches(dev, 1)[0]
    assert bool(train_step(m, make_optimizer(m, m.cfg), x).isfinite())
    f = m.blocks[0].ffn
    h = seeded((2, 70, 64), 5, torch.float32, dev).requires_grad_()
    dy = seeded((2, 70, 64), 6, torch.float32, dev)
    leaves = [h, *f.parameters()]
    ref = torch.autograd.grad(f(h), leaves, dy)
    again = torch.autograd.grad(torch.utils.checkpoint.checkpoint(f, h, use_reentrant=False), leaves, dy)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.to(dev)):
        away = torch.autograd.grad(f(h), leaves, dy)
    for a, b, c in zip(ref, again, away):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_inputs_changed_in_place_are_noticed(dev):
    x, w = seeded((6, 16), 7, torch.float32, dev), seeded((20, 16), 8, torch.float32, dev).requires_grad_()
    target = torch.arange(6, device=dev)
    loss = linear_cross_entropy(x, w, target)
    target[0] = 3
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(loss, w)


@pytest.mark.parametrize("dtype,keep", [(torch.bfloat16, 1), (torch.bfloat16, 2), (torch.float32, 1)])
def test_opcheck_gated_ffn(dev, dtype, keep):
    x, w_in, w_down = (seeded(s, 10 + i, dtype, dev).requires_grad_() for i, s in
                       enumerate(((2, 9, 16), (24, 16), (16, 12))))
    torch.library.opcheck(torch.ops.pnfx.gated_ffn.default, (x, w_in, w_down, 0, keep))
    a = [t.detach() for t in (x, w_in, w_down)]
    torch.library.opcheck(torch.ops.pnfx.gated_ffn.default, (*a, 1, 0))
    y, gu, sc = torch.ops.pnfx.gated_ffn(*a, 0, keep)
    torch.library.opcheck(torch.ops.pnfx.gated_ffn_bwd.default,
                          (torch.randn_like(y), *a, gu, sc, 0, keep, [True, False, True]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("reduction", [0, 2])
def test_opcheck_linear_xent(dev, dtype, reduction):
    x, w = (seeded(s, 20 + i, dtype, dev).requires_grad_() for i, s in enumerate(((2, 9, 16), (24, 16))))
    t = torch.randint(0, 24, (2, 9), generator=torch.Generator().manual_seed(0)).to(dev)
    torch.library.opcheck(torch.ops.pnfx.linear_xent.default, (x, w, t, 5, reduction))
    a = [v.detach() for v in (x, w)]
    loss, rows, lse = torch.ops.pnfx.linear_xent(*a, t, 5, reduction)
    torch.library.opcheck(torch.ops.pnfx.linear_xent_bwd.default,
                          (torch.ones_like(loss), *a, t, rows, lse, 5, reduction, [True, True]))


def test_compiled_block_and_loss(dev):
    """torch.compile traces block and loss as one graph, forward and backward (AOTAutograd's eager backend)."""
    from paper_01_anti_decoy_pnfirtau_amd.wikilm import GatedFFN

    f = GatedFFN(32, 40, "gelu", checkpoint="e4m3").to(dev).bfloat16()
    w = seeded((50, 32), 30, torch.bfloat16, dev).requires_grad_()
    x, target = seeded((3, 20, 32), 31, torch.bfloat16, dev), torch.randint(0, 50, (3, 20)).to(dev)

    def step(x, target):
        return linear_cross_entropy(x + f(x), w, target)

    compiled = torch.compile(step, backend="aot_eager", fullgraph=True)
    leaves = [w, *f.parameters()]
    for _ in range(2):
        got, ref = compiled(x, target), step(x, target)
        assert torch.equal(got, ref)
        for a, b in zip(torch.autograd.grad(got, leaves), torch.autograd.grad(ref, leaves)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("T", [1, 40, 300])
def test_threads_and_streams_at_once(dev, T):
    """Four threads with a stream each, inference and training calls mixed: every result is that of a call alone."""
    import threading

    D, Fd, V = 64, 96, 700
    w_in, w_down = seeded((2 * Fd, D), 32, torch.bfloat16, dev, 0.1), seeded((D, Fd), 33, torch.bfloat16, dev, 0.1)
    w = seeded((V, D), 34, torch.bfloat16, dev)

    def run(i):
        x = seeded((T, D), 40 + i, torch.bfloat16, dev).requires_grad_()
        target = torch.arange(T, device=dev) * (i + 1) % V
        with torch.no_grad():
            y = gated_ffn(x, w_in, w_down)
        loss = linear_cross_entropy(gated_ffn(x, w_in, w_down), w, target)
        return [y, loss.detach(), torch.autograd.grad(loss, x)[0]]

    ref = [run(i) for i in range(4)]
    torch.cuda.synchronize()
    got = [None] * 4

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                got[i] = run(i)
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(got, ref):
        assert all(torch.equal(u, v) for u, v in zip(a, b))
