"""The language model that consumes the pn_fir_tau attention path, and its training step.

Mirrors the reference's WikiText-2 model and step (``experiments/exp4_wikitext2_lm.py``):

* ``Block``   :183-201 -- pre-LN residual block: x + drop(attn(ln1 x)), then
  x + ffn(ln2 x) with ffn = Linear -> GELU -> Linear -> Dropout;
* ``WikiLM``  :203-247 -- token + learned position embeddings, ``n_layers`` blocks with the
  chosen attention module, final LayerNorm and a head tied to the token embedding;
* ``train_step`` :334-348 -- zero_grad, bf16 autocast forward, next-token cross-entropy,
  backward, AdamW (betas 0.9/0.95).

Beside the reference's model, ``WikiLMConfig`` offers two choices that it does not have: a gated
feed-forward block (``ffn="swiglu"`` or ``"geglu"``: ``GatedFFN``, whose activations may be kept in
8 bits) and the loss without materialised logits (``fused_loss``); and a model can answer, which the
reference's does not: ``generate`` continues prompts token by token over 8-bit caches, ``Decoder`` is its engine.

``GraphedStep`` captures that whole step (including the optimizer update) in one HIP graph,
as the reference's ``experiments/exp4c_cuda_graphs.py:81-108`` does for the attention stack:
the eager stack is launch-bound at these sizes.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch
import torch.nn as nn
import torch.nn.functional as F

from .hip_cache import KVCache, sample_tokens, whole_numbers
from .hip_lm import gated_ffn, linear_cross_entropy
from .pnfirtau_attention import PnFirConfig, PnFirTauFlashMHA, PnFirTauMHA, PnFirTauTritonMHA

ATTENTION = {
    "pn_fir_tau": PnFirTauMHA,
    "pn_fir_tau_triton": PnFirTauTritonMHA,
    "pn_fir_tau_flash": PnFirTauFlashMHA,
}


GATED_FFN = {"swiglu": "silu", "geglu": "gelu"}  # WikiLMConfig.ffn: the gate's activation


@dataclass
class WikiLMConfig:
    """Model shape and optimiser settings (defaults of experiments/exp4_wikitext2_lm.py:67-88).

    ``ffn``: "gelu", the reference's two-layer FFN, or a gated one, "swiglu" or "geglu" (d_ff columns
    each for the gate and the up projection); ``ffn_checkpoint``: how a gated FFN keeps its
    projections for the backward pass, "full" or "e4m3" (hip_lm.gated_ffn: the latter for training
    under bf16 autocast).  ``fused_loss``: lm_loss computes the loss with hip_lm.linear_cross_entropy
    instead of materialised logits (faster in bf16; in fp32 it saves their memory, not time)."""

    d_model: int = 64
    n_heads: int = 4
    n_layers: int = 6
    d_ff: int = 256
    max_seq: int = 256
    lr: float = 5e-4
    weight_decay: float = 0.1
    dropout: float = 0.1
    p: float = 10.0
    silence_gamma: float = 0.5
    tau_init: float = 0.0
    fir_k: int = 7
    ffn: str = "gelu"
    ffn_checkpoint: str = "full"
    fused_loss: bool = False


class GatedFFN(nn.Module):
    """Bias-free gated feed-forward block with dropout on its output: ``gate_up.weight`` holds the gate's
    d_ff rows, then the up projection's (hip_lm.gated_ffn)."""

    def __init__(self, d_model: int, d_ff: int, activation: str = "silu", dropout: float = 0.0,
                 checkpoint: str = "full"):
        super().__init__()
        self.gate_up = nn.Linear(d_model, 2 * d_ff, bias=False)
        self.down = nn.Linear(d_ff, d_model, bias=False)
        self.drop = nn.Dropout(dropout)
        self.activation, self.checkpoint = activation, checkpoint

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return self.drop(gated_ffn(x, self.gate_up.weight, self.down.weight, self.activation,
                                   self.checkpoint))


class Block(nn.Module):
    """Pre-LN residual block (experiments/exp4_wikitext2_lm.py:183-201)."""

    def __init__(self, d_model: int, attn: nn.Module, dropout: float, d_ff: int, ffn: str = "gelu",
                 ffn_checkpoint: str = "full"):
        super().__init__()
        self.ln1 = nn.LayerNorm(d_model)
        self.attn = attn
        self.ln2 = nn.LayerNorm(d_model)
        if ffn in GATED_FFN:
            self.ffn = GatedFFN(d_model, d_ff, GATED_FFN[ffn], dropout, ffn_checkpoint)
        elif ffn == "gelu":
            self.ffn = nn.Sequential(
                nn.Linear(d_model, d_ff), nn.GELU(), nn.Linear(d_ff, d_model), nn.Dropout(dropout)
            )
        else:
            raise ValueError(f"Unknown ffn: {ffn}")
        self.drop = nn.Dropout(dropout)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        x = x + self.drop(self.attn(self.ln1(x)))
        return x + self.ffn(self.ln2(x))

    def forward_cached(self, x: torch.Tensor, cache: KVCache, start, counts=None) -> torch.Tensor:
        x = x + self.attn.forward_cached(self.ln1(x), cache, start, counts)
        return x + self.ffn(self.ln2(x))


class WikiLM(nn.Module):
    """Decoder-only LM with pn_fir_tau attention (experiments/exp4_wikitext2_lm.py:203-247).

    ``variant`` picks the attention module: ``pn_fir_tau`` (eager), ``pn_fir_tau_triton``
    (row-fused scores) or ``pn_fir_tau_flash`` (flash).  Parameters are created in the
    reference's order, so the same seed gives the same initial weights for every variant.
    """

    def __init__(self, vocab: int, cfg: WikiLMConfig, variant: str = "pn_fir_tau_flash"):
        super().__init__()
        if variant not in ATTENTION:
            raise ValueError(f"Unknown variant: {variant}")
        self.cfg = cfg
        self.variant = variant
        self.embed = nn.Embedding(vocab, cfg.d_model)
        self.pos = nn.Embedding(cfg.max_seq, cfg.d_model)
        self.drop = nn.Dropout(cfg.dropout)
        acfg = PnFirConfig(
            d_model=cfg.d_model, n_heads=cfg.n_heads, p=cfg.p, silence_gamma=cfg.silence_gamma,
            tau_init=cfg.tau_init, fir_k=cfg.fir_k, dropout=cfg.dropout, causal_mask=True,
            bias=False,
        )
        self.blocks = nn.ModuleList(
            Block(cfg.d_model, ATTENTION[variant](acfg), cfg.dropout, cfg.d_ff, cfg.ffn,
                  cfg.ffn_checkpoint)
            for _ in range(cfg.n_layers)
        )
        self.ln_f = nn.LayerNorm(cfg.d_model)
        self.head = nn.Linear(cfg.d_model, vocab, bias=False)
        self.head.weight = self.embed.weight

    def hidden(self, idx: torch.Tensor) -> torch.Tensor:
        """The rows [B, N, d_model] that the head projects to logits."""
        _, n = idx.shape
        pos = torch.arange(n, device=idx.device).unsqueeze(0)
        h = self.drop(self.embed(idx) + self.pos(pos))
        for blk in self.blocks:
            h = blk(h)
        return self.ln_f(h)

    def forward(self, idx: torch.Tensor) -> torch.Tensor:
        return self.head(self.hidden(idx))

    def new_caches(self, batch: int, max_len: int | None = None, **kwargs) -> list[KVCache]:
        """One empty cache for each layer, for sequences of up to max_len tokens (at most, and by default, the model's
        max_seq), with one table."""
        if max_len is not None and max_len > self.cfg.max_seq:
            raise ValueError(f"new_caches: {max_len} tokens of a model of {self.cfg.max_seq}")
        caches: list[KVCache] = []
        for blk in self.blocks:
            shared = {"table": caches[0].table, "pages": caches[0].k.shape[0]} if caches else {}
            caches.append(blk.attn.new_cache(batch, max_len or self.cfg.max_seq, **{**kwargs, **shared}))
        return caches

    def hidden_cached(self, idx: torch.Tensor, caches: list[KVCache], start: int | torch.Tensor,
                      counts: torch.Tensor | None = None) -> torch.Tensor:
        """As ``hidden``, of the tokens idx [B, N] that follow those in the caches (which they join): positions start ..
        start + N - 1, of which a sequence has ``counts``.  In evaluation mode, under torch.no_grad().  The model has no
        positions from max_seq on: ValueError where the host knows, otherwise NaN for those tokens."""
        most, known = self.cfg.max_seq, not torch.is_tensor(start) and counts is None
        if known and start + idx.shape[1] > most:
            raise ValueError(f"hidden_cached: tokens {start} .. {start + idx.shape[1] - 1} of a model of {most}")
        pos = torch.arange(idx.shape[1], device=idx.device) + (start[:, None] if torch.is_tensor(start) else start)
        h = self.embed(idx) + self.pos(pos.clamp(0, most - 1))
        if not known and any(c.capacity > most for c in caches):  # whole pages; beyond them the cache gives NaN
            h = h.masked_fill((pos >= most)[..., None], torch.nan)
        for blk, cache in zip(self.blocks, caches):
            h = blk.forward_cached(h, cache, start, counts)
        return self.ln_f(h)


def zipf_tokens(batch: int, seq: int, vocab: int, seed: int, s: float = 1.1) -> torch.Tensor:
    """Synthetic token ids [batch, seq] ~ Zipf(s) truncated to [0, vocab) by rejection,
    seeded on the CPU (the benchmark LM workload: no dataset is fetched)."""
    import numpy as np

    rng = np.random.default_rng(seed)
    need, out = batch * seq, []
    while need > 0:
        z = rng.zipf(s, size=2 * need) - 1
        z = z[z < vocab][:need]
        out.append(z)
        need -= len(z)
    return torch.from_numpy(np.concatenate(out).reshape(batch, seq).astype(np.int64))


def make_optimizer(model: nn.Module, cfg: WikiLMConfig, capturable: bool = False,
                   fused: bool | None = None):
    """AdamW as the reference builds it (experiments/exp4_wikitext2_lm.py:326-328).

    ``fused=True`` selects torch's single-kernel AdamW (same update rule); with
    ``capturable=True`` it is the cheapest optimizer step to capture in a graph.
    """
    return torch.optim.AdamW(model.parameters(), lr=cfg.lr, betas=(0.9, 0.95),
                             weight_decay=cfg.weight_decay, capturable=capturable, fused=fused)


def lm_loss(model: nn.Module, x: torch.Tensor, amp: bool) -> torch.Tensor:
    """Next-token cross-entropy over the sequence, under bf16 autocast when ``amp``; without the logits
    where the model's config has ``fused_loss`` (each sequence's last row, which has no next token, is
    ignored there).  The context keeps no casts of the weights: a caller's autocast around it would keep them over
    optimizer steps, and beyond a captured step's memory."""
    vocab = model.head.weight.shape[0]
    with torch.autocast(device_type=x.device.type, dtype=torch.bfloat16, enabled=amp, cache_enabled=False):
        if getattr(getattr(model, "cfg", None), "fused_loss", False):
            target = torch.cat([x[:, 1:], x.new_full((x.shape[0], 1), -100)], 1)
            return linear_cross_entropy(model.hidden(x), model.head.weight, target)
        logits = model(x)
        return F.cross_entropy(logits[:, :-1].reshape(-1, vocab), x[:, 1:].reshape(-1))


def train_step(model: nn.Module, opt: torch.optim.Optimizer, x: torch.Tensor,
               amp: bool = True) -> torch.Tensor:
    """One step of experiments/exp4_wikitext2_lm.py:334-348; returns the loss (a tensor)."""
    opt.zero_grad(set_to_none=True)
    loss = lm_loss(model, x, amp)
    loss.backward()
    opt.step()
    return loss.detach()


class GraphedStep:
    """The training step of ``train_step`` captured once as a HIP graph and replayed.

    Gradients are cleared by a fill kernel inside the graph (``zero_grad`` with
    ``set_to_none=False``) rather than by dropping the tensors, so the captured addresses stay
    valid; the optimizer must be built with ``capturable=True`` and have no state yet.  ``x``
    is a static input: copy new tokens into it before ``replay``.  The loss of the last replay
    is ``self.loss``.

    Construction runs ``warmup`` real steps on ``x`` (the allocator and the optimizer's state
    must exist before capture), then puts every parameter and buffer back and zeroes the
    optimizer state in place (for Adam-type optimizers a zero state, step count included, is
    the fresh state): the first ``replay`` is the model's first training step.
    """

    def __init__(self, model: nn.Module, opt: torch.optim.Optimizer, x: torch.Tensor,
                 amp: bool = True, warmup: int = 3):
        self.model, self.opt, self.x, self.amp = model, opt, x, amp
        if any(len(st) for st in opt.state.values()):
            raise ValueError("GraphedStep: the optimizer already has state")
        saved = [t.detach().clone() for t in list(model.parameters()) + list(model.buffers())]
        with torch.cuda.device(x.device):  # a capture is of the current device's streams
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                for _ in range(warmup):
                    self._step()
            torch.cuda.current_stream().wait_stream(side)
            self.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.graph):
                self.loss = self._step()
        # capture records the step without running it: undo the warm-up steps in place, so
        # the captured addresses stay the live ones
        with torch.no_grad():
            for t, s in zip(list(model.parameters()) + list(model.buffers()), saved):
                t.copy_(s)
            for st in opt.state.values():
                for v in st.values():
                    if torch.is_tensor(v):
                        v.zero_()

    def _step(self) -> torch.Tensor:
        self.opt.zero_grad(set_to_none=False)
        loss = lm_loss(self.model, self.x, self.amp)
        loss.backward()
        self.opt.step()
        return loss.detach()

    def replay(self) -> torch.Tensor:
        self.graph.replay()
        return self.loss


class Decoder:
    """Continues sequences of one model, a token of each at a time, over 8-bit caches.

    ``prefill`` takes the prompts, ``step`` draws the next token of every sequence and takes it in; where the sequences
    are stands on the device, so that with ``graph`` a step is one captured HIP graph.  ``settings``: sample_tokens'
    (values, or tensors [B] whose contents may change between steps).  The model must be in evaluation mode.
    ``amp``: bf16 autocast."""

    def __init__(self, model: WikiLM, batch: int, max_len: int | None = None, amp: bool = False, graph: bool = False,
                 **settings):
        if model.training:
            raise ValueError("Decoder: the model is in training mode")
        self.model, self.amp, self.graph, self.settings = model, amp, graph, settings
        self.max_len = model.cfg.max_seq if max_len is None else max_len
        if self.max_len > model.cfg.max_seq:
            raise ValueError(f"Decoder: {self.max_len} tokens of a model of {model.cfg.max_seq}")
        dev, dtype = model.embed.weight.device, model.embed.weight.dtype
        self.caches = model.new_caches(batch, self.max_len, dtype=torch.bfloat16 if amp else dtype)
        self.start = torch.zeros(batch, dtype=torch.int32, device=dev)
        self.rows = torch.zeros(batch, model.cfg.d_model, dtype=dtype, device=dev)  # before the head, of the last tokens
        self.u = torch.zeros(batch, device=dev)
        self.token = torch.zeros(batch, dtype=torch.int64, device=dev)
        self.most = 0  # tokens of the longest sequence
        self._captured = None

    def _autocast(self):
        """bf16 where ``amp``, without the cache of cast weights: inside a caller's autocast it outlives this context, and
        a captured step would read its copies from outside the graph, after they are freed; they would not follow
        weights that change in place either."""
        return torch.autocast(self.rows.device.type, torch.bfloat16, enabled=self.amp, cache_enabled=False)

    def _run(self, idx, start, counts=None):
        with torch.no_grad(), self._autocast():
            return self.model.hidden_cached(idx, self.caches, start, counts)

    def prefill(self, prompt: torch.Tensor, lengths: torch.Tensor | None = None) -> None:
        """Begins anew with the prompts [B, N], of which sequence b has lengths[b] tokens (null: N).  A length outside 1
        .. N is a ValueError where it is on the host; nothing waits for the device to look at one there: such a sequence
        gets -1 for every token."""
        B, N = prompt.shape
        if not 0 < N <= self.max_len or B != len(self.start):
            raise ValueError(f"Decoder: prompts {tuple(prompt.shape)} for {len(self.start)} sequences of {self.max_len}")
        counts = whole_numbers("lengths", lengths, B)
        if counts is None:
            h = self._run(prompt, 0)
            self.rows.copy_(h[:, -1])
            self.start.fill_(N)
        else:
            bad = (counts < 1) | (counts > N)
            if not bad.is_cuda and bad.any():
                raise ValueError(f"Decoder: lengths {lengths.tolist()} of prompts of {N} tokens")
            counts, bad = counts.to(self.start.device), bad.to(self.start.device)
            h = self._run(prompt, 0, counts)
            last = (counts.clamp(1, N).long() - 1)[:, None, None].expand(B, 1, h.shape[2])
            self.rows.copy_(h.gather(1, last)[:, 0].masked_fill(bad[:, None], torch.nan))
            self.start.copy_(counts.masked_fill(bad, -(1 << 30)))  # below zero at every step: NaN from the caches
        self.most = N

    def _step(self) -> None:
        with torch.no_grad(), self._autocast():
            token = sample_tokens(self.model.head(self.rows), self.u, **self.settings)
        h = self._run(token.clamp(min=0)[:, None], self.start)  # -1: a row of NaN has no token
        self.rows.copy_(h[:, 0])
        self.start += 1
        self.token.copy_(token)

    def step(self, u: torch.Tensor) -> torch.Tensor:
        """The next token of each sequence, drawn by u [B] in [0, 1); overwritten by the next call.  -1: a sequence whose
        logits hold a NaN."""
        if not self.most:
            raise ValueError("Decoder: no prompts yet")
        if u.shape != self.u.shape:
            raise ValueError(f"Decoder: u has shape {tuple(u.shape)}, not {tuple(self.u.shape)}")
        if self.most + 1 > self.max_len:
            raise ValueError(f"Decoder: sequences of {self.max_len} tokens are full")
        self.most += 1
        self.u.copy_(u)
        if not (self.graph and self.u.is_cuda):
            self._step()
            return self.token
        if self._captured is None:
            with torch.cuda.device(self.u.device):  # a capture is of the current device's streams
                self._capture()
        self._captured.replay()
        return self.token

    def _capture(self) -> None:
        # the warm-up runs on what a step overwrites: the caches' next token, written again by the replay, and state
        # that is put back
        saved = self.rows.clone(), self.start.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            self._step()
            self.rows.copy_(saved[0]), self.start.copy_(saved[1])
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            self._step()
        self._captured = graph


def generate(model: WikiLM, prompt: torch.Tensor, max_new: int, lengths: torch.Tensor | None = None,
             u: torch.Tensor | None = None, generator: torch.Generator | None = None, amp: bool = False,
             graph: bool = False, **settings) -> torch.Tensor:
    """max_new tokens [B, max_new] that follow the prompts [B, N] (sequence b has lengths[b] of the N), drawn by u
    [B, max_new] (by default from ``generator``) with sample_tokens' ``settings``."""
    B, N = prompt.shape
    if u is None:
        dev = prompt.device if generator is None else generator.device
        u = torch.rand(B, max_new, generator=generator, device=dev).to(prompt.device)
    if u.shape != (B, max_new):
        raise ValueError(f"generate: u has shape {tuple(u.shape)}, not {(B, max_new)}")
    dec = Decoder(model, B, N + max_new, amp=amp, graph=graph, **settings)
    dec.prefill(prompt, lengths)
    return torch.stack([dec.step(u[:, i]).clone() for i in range(max_new)], 1) if max_new else prompt.new_empty(B, 0)
