"""The gated feed-forward block and the vocabulary cross entropy: the calls whose time is measured.

Kinds of case:

* ``ffn``   the gated feed-forward block ``y = (act(x Wg^T) * (x Wu^T)) Wd^T`` on rows ``x [T, D]``, with
            ``w_in [2 F, D]`` (the rows of Wg, then those of Wu) and ``w_down [D, F]``: inference, or a
            training call (y and the gradients of x, w_in and w_down for a given dy) that keeps the two
            projections either in the operands' type (``full``) or, of bf16 rows, in 8 bits
            (``e4m3``);
* ``xent``  softmax cross entropy of the logits ``x W^T`` (``x [T, D]``, ``W [V, D]``) against the target
            tokens, some rows of which are padding: the loss alone, or the loss with the gradients of x
            and W.

In 8 bits a projection's row is held in blocks of 32 columns (the last may be shorter), each with the
smallest power of two s for which no |value| / s is above 448, the largest e4m3 number; the values over s
are rounded to e4m3, ties to even, and the backward pass computes with what these stand for.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
IGNORE = -100
BLOCK = 32  # columns that share a scale in 8 bits
SEQ = 512   # rows of one sequence, for the padding of the cross entropy's rows


def _ffn(name, T, D, F, mode="train", act="silu", keep="full", dtype="bf16"):
    return dict(name=name, kind="ffn", T=T, D=D, F=F, mode=mode, act=act, keep=keep, dtype=dtype)


def _xent(name, T, D, V, mode="train", reduction="mean", pad=0.0, dtype="bf16"):
    return dict(name=name, kind="xent", T=T, D=D, V=V, mode=mode, reduction=reduction, pad=pad,
                dtype=dtype)


def listed():
    return [
        # Serving, one sequence: a single token's block, where the weights' bytes and the launches count.
        _ffn("ffn_token", 1, 1024, 4096, mode="infer"),
        # Serving a batch: one token for each of 40 sequences.
        _ffn("ffn_batch", 40, 2048, 5632, mode="infer"),
        # A prompt's rows in inference.
        _ffn("ffn_prompt", 4096, 1024, 4096, mode="infer", act="gelu"),
        # The benchmark's language model (32 sequences of 512 tokens, D = 256, d_ff = 1024) in training.
        _ffn("ffn_train", 16384, 256, 1024),
        # A wide model in training, its activations kept in 8 bits.
        _ffn("ffn_train_8bit", 8192, 2048, 8192, keep="e4m3"),
        # Sizes that fit no tile, chunk or block.
        _ffn("ffn_ragged", 1531, 250, 666, act="gelu"),
        # Full precision (parity runs with reduced precision switched off).
        _ffn("ffn_f32", 4096, 256, 1024, dtype="f32"),
        # The benchmark's language model: its head's loss over the vocabulary in training.
        _xent("xent_lm", 16384, 256, 33278, pad=0.02),
        # The reference's small model: a narrow head, so that the exponentials count and not the products.
        _xent("xent_narrow", 16384, 64, 23168),
        # A wide model with a large vocabulary, a fifth of its rows padding: the largest call.
        _xent("xent_large", 8192, 2048, 65536, pad=0.2),
        # Scoring a short text: every token's loss, no gradient, sizes that fit no tile.
        _xent("xent_score", 333, 1000, 50257, mode="score", reduction="none"),
        # Full precision.
        _xent("xent_f32", 2048, 256, 8191, reduction="sum", pad=0.1, dtype="f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size spread over its logarithm: two in three a multiple of 16, the others as they come."""
    n = _log(rng, lo, hi)
    return max(lo, n // 16 * 16) if rng.random() < 2 / 3 else n


def draw(rng):
    dtype = "f32" if rng.random() < 0.2 else "bf16"
    most = 2e11 if dtype == "f32" else 2e12  # operations: no more than the largest listed case has
    if rng.random() < 0.5:
        mode = rng.choice(["infer", "train", "train"])
        T = _log(rng, 1, 256) if mode == "infer" and rng.random() < 0.6 else _size(rng, 64, 16384)
        D = _size(rng, 32, 4096)
        F = _size(rng, max(32, D), 4 * D)
        while work(dict(kind="ffn", T=T, D=D, F=F, mode=mode, dtype=dtype))["flops"] > most:
            T = T // 2 + 1
        return dict(kind="ffn", T=T, D=D, F=F, mode=mode, act=rng.choice(["silu", "gelu"]),
                    keep=rng.choice(["full", "e4m3"]) if (mode, dtype) == ("train", "bf16") else "full",
                    dtype=dtype)
    mode = rng.choice(["score", "train", "train"])
    T = _log(rng, 1, 256) if mode == "score" and rng.random() < 0.4 else _size(rng, 64, 16384)
    D = _size(rng, 32, 2048)
    V = _size(rng, 256, 131072)
    pad = rng.choice([0.0, 0.0, 0.05, 0.4])
    while work(dict(kind="xent", T=T, D=D, V=V, mode=mode, pad=pad, dtype=dtype))["flops"] > most:
        T, V = T // 2 + 1, V // 2 + 1
    return dict(kind="xent", T=T, D=D, V=V, mode=mode,
                reduction=rng.choice(["none", "sum", "mean"]) if mode == "score" else
                rng.choice(["sum", "mean", "mean"]), pad=pad, dtype=dtype)


def work(case):
    T, D = case["T"], case["D"]
    es = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "ffn":
        F = case["F"]
        if case["mode"] == "infer":  # x, the weights; y
            return {"bytes": es * (2 * T * D + 3 * F * D), "flops": 6.0 * T * D * F}
        # x, dy, the weights; y and the gradients of x and the weights
        return {"bytes": es * (4 * T * D + 6 * F * D), "flops": 18.0 * T * D * F}
    V, kept = case["V"], max(1.0, T * (1 - case["pad"]))
    if case["mode"] == "score":  # x, W, targets; losses
        return {"bytes": es * (kept * D + V * D) + 12 * T, "flops": 2.0 * kept * D * V}
    # x, W, targets; the gradients of x and W
    return {"bytes": es * (kept * D + T * D + 2 * V * D) + 8 * T, "flops": 6.0 * kept * D * V}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    T, D = case["T"], case["D"]

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dt)

    s = dict(case, x=normal(T, D))  # rows behind a layer norm
    train = case["mode"] == "train"
    if case["kind"] == "ffn":
        F = case["F"]
        s["w_in"], s["w_down"] = normal(2 * F, D, std=1.5 * D ** -0.5), normal(D, F, std=F ** -0.5)
        if train:
            s["dy"] = normal(T, D, std=0.1)
            for n in ("x", "w_in", "w_down"):
                s[n].requires_grad_()
        return s
    s["w"] = normal(case["V"], D, std=2 * D ** -0.5)
    u = torch.rand(T, generator=g, device="cuda", dtype=torch.float64)
    target = (case["V"] * u ** 4).long().clamp_(max=case["V"] - 1)  # frequent tokens first
    if case["pad"]:  # the ends of the sequences, uneven
        n = -(-T // SEQ)
        ends = SEQ * (1 - 2 * case["pad"] * torch.rand(n, generator=g, device="cuda"))
        row = torch.arange(T, device="cuda")
        target = torch.where(row % SEQ < ends[row // SEQ], target, IGNORE)
    s["target"] = target
    if train:
        for n in ("x", "w"):
            s[n].requires_grad_()
    return s


# ------------------------------------------------------------------------------- plain forms
def _e4m3(v):
    """What rows v [T, n] stand for after a round trip through 8 bits."""
    T, n = v.shape
    b = torch.zeros(T, -(-n // BLOCK) * BLOCK, dtype=v.dtype, device=v.device)
    b[:, :n] = v
    b = b.view(T, -1, BLOCK)
    top = b.abs().amax(2, keepdim=True)
    m, e = torch.frexp(top / 448)  # top / 448 = m 2^e, m in [1/2, 1): s = 2^e, or 2^(e-1) where m is 1/2
    one = torch.ones_like(top)
    s = torch.ldexp(one, torch.where(m == 0.5, e - 1, e).clamp(min=-126))
    r = b / s
    _, q = torch.frexp(r)
    step = torch.ldexp(one, (q - 4).clamp(min=-9))  # four significant bits, 2^-9 below 2^-6
    return ((r / step).round() * step * s).view(T, -1)[:, :n]


def _act(v, act):
    """act(v) and its derivative."""
    if act == "silu":
        p = 1 / (1 + torch.exp(-v))
        return v * p, p * (1 + v * (1 - p))
    p = 0.5 * (1 + torch.erf(v * 0.5 ** 0.5))
    return v * p, p + v * torch.exp(-0.5 * v * v) * (2 * math.pi) ** -0.5


def _plain_ffn(s):
    dt = s["x"].dtype
    x, w_in, w_down = (s[n].detach().float() for n in ("x", "w_in", "w_down"))
    F = s["F"]
    gu = x @ w_in.t()
    y = (_act(gu[:, :F], s["act"])[0] * gu[:, F:]) @ w_down.t()
    if s["mode"] == "infer":
        return y.to(dt)
    g, u = gu[:, :F], gu[:, F:]
    if s["keep"] == "e4m3":
        g, u = _e4m3(g), _e4m3(u)
    dy = s["dy"].float()
    a, da = _act(g, s["act"])
    dh = dy @ w_down
    dgu = torch.cat([dh * u * da, dh * a], 1)
    return [t.to(dt) for t in (y, dgu @ w_in, dgu.t() @ x, dy.t() @ (a * u))]


def _plain_xent(s):
    dt = s["x"].dtype
    x, w, target = s["x"].detach().float(), s["w"].detach().float(), s["target"]
    kept = target != IGNORE
    at = torch.where(kept, target, 0)[:, None]
    z = x @ w.t()
    z = z - z.amax(1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    rows = torch.where(kept, (torch.log(total) - z.gather(1, at))[:, 0], 0.0)
    scale = 1 / kept.sum() if s["reduction"] == "mean" else 1.0
    loss = rows if s["reduction"] == "none" else (rows.double().sum() * scale).float()
    if s["mode"] == "score":
        return loss
    d = e / total
    d.scatter_add_(1, at, -torch.ones_like(total))
    d = d * (kept[:, None] * scale)
    return [loss, (d @ w).to(dt), (d.t() @ x).to(dt)]


# ------------------------------------------------------------------------- the framework's calls
def _own_ffn(s):
    from paper_01_anti_decoy_pnfirtau_amd import gated_ffn

    y = gated_ffn(s["x"], s["w_in"], s["w_down"], activation=s["act"], checkpoint=s["keep"])
    if s["mode"] == "infer":
        return y
    return [y.detach(), *torch.autograd.grad(y, (s["x"], s["w_in"], s["w_down"]), s["dy"])]


def _own_xent(s):
    from paper_01_anti_decoy_pnfirtau_amd import linear_cross_entropy

    loss = linear_cross_entropy(s["x"], s["w"], s["target"], ignore_index=IGNORE,
                                reduction=s["reduction"])
    if s["mode"] == "score":
        return loss
    return [loss.detach(), *torch.autograd.grad(loss, (s["x"], s["w"]))]


def run(state):
    if state["kind"] == "ffn":
        return _own_ffn(state) if own else _plain_ffn(state)
    return _own_xent(state) if own else _plain_xent(state)


# ------------------------------------------------------------------------------- in 64 bits
def _exact_8bit(v):
    """Row by block: the e4m3 numbers nearest to v / 2^k, times 2^k, from the format's definition."""
    pad = -v.shape[1] % BLOCK
    blocks = torch.nn.functional.pad(v, (0, pad)).unflatten(1, (-1, BLOCK))
    top = blocks.abs().max(2, keepdim=True).values
    k = torch.ceil(torch.log2((top / 448).clamp(min=2.0 ** -126)))
    k = torch.where(top > 448 * 2 ** k, k + 1, k)
    k = torch.where((top <= 448 * 2 ** (k - 1)) & (k > -126), k - 1, k)
    r = blocks * 2 ** -k
    binade = torch.floor(torch.log2(r.abs().clamp(min=2.0 ** -6)))
    binade = torch.where(r.abs().clamp(min=2.0 ** -6) < 2 ** binade, binade - 1, binade)
    return (torch.round(r * 2 ** (3 - binade)) * 2 ** (binade - 3 + k)).flatten(1)[:, :v.shape[1]]


def _exact_act(v, act):
    if act == "silu":
        return v * torch.sigmoid(v), torch.sigmoid(v) + v * torch.sigmoid(v) * torch.sigmoid(-v)
    density = torch.exp(-v.square() / 2) / math.sqrt(2 * math.pi)
    cdf = torch.special.ndtr(v)
    return v * cdf, cdf + v * density


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].detach().double()
    if case["kind"] == "ffn":
        wg, wu = s["w_in"].detach().double().chunk(2)
        wd = s["w_down"].detach().double()
        g, u = x.matmul(wg.mT), x.matmul(wu.mT)
        y = (_exact_act(g, case["act"])[0] * u).matmul(wd.mT)
        if case["mode"] == "infer":
            return y
        if case["keep"] == "e4m3":
            g, u = _exact_8bit(g), _exact_8bit(u)
        dy = s["dy"].double()
        a, slope = _exact_act(g, case["act"])
        dh = dy.matmul(wd)
        dg, du = dh * slope * u, dh * a
        return [y, dg.matmul(wg) + du.matmul(wu), torch.cat([dg.mT.matmul(x), du.mT.matmul(x)]),
                dy.mT.matmul(a * u)]
    w = s["w"].detach().double()
    keep = (s["target"] != IGNORE).nonzero()[:, 0]
    rows, to = x[keep], s["target"][keep]
    logp = torch.log_softmax(rows.matmul(w.mT), 1)
    each = -logp[torch.arange(len(to), device=to.device), to]
    if case["reduction"] == "none":
        loss = torch.zeros(case["T"], dtype=torch.float64, device=x.device).index_copy(0, keep, each)
    else:
        loss = each.sum() / (len(to) if case["reduction"] == "mean" else 1)
    if case["mode"] == "score":
        return loss
    d = logp.exp_()
    d[torch.arange(len(to), device=to.device), to] -= 1
    if case["reduction"] == "mean":
        d /= len(to)
    dx = torch.zeros_like(x).index_copy_(0, keep, d.matmul(w))
    return [loss, dx, d.mT.matmul(rows)]
