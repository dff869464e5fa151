"""Answering with a trained model: the 8-bit key and value cache, attention over it, the draw of the next token.

================================  ==================================================================
``KVCache.append``                keys behind the causal FIR and values, rounded to 8 bits as they are written
``KVCache.read``                  the cache as dense keys and values
``cached_attention``              pn_fir_tau attention (p = 10, peak gate) of the last tokens over the cache
``sample_tokens``                 temperature, top-k, top-p and min-p from given random numbers
================================  ==================================================================

None has a counterpart in the reference, whose attention is over dense keys of equal length
(src/triton_pnfirtau.py:814-983) and which does not generate.  GPU tensors, bf16 or fp32, run the HIP kernels
(``pnfx::cache_append``, ``cache_read``, ``cached_attn``, ``sample_tokens``), none of which waits for the device; CPU
tensors the same in torch operations.  None has gradients: writing and attention raise where one would be recorded, or forward
mode's tangent carried.
"""
from __future__ import annotations

import functools
import math
import operator
from dataclasses import dataclass

import torch
import torch.nn.functional as F
from torch.autograd import forward_ad

BLOCK = 16         # tokens that share a scale
RAW = 16           # keys before the FIR that are kept of each sequence
LOWEST = -100      # smallest scale: 2^LOWEST
MAX_HEAD_DIM = 256
MAX_TAPS = 16
MAX_PAGE, MAX_CAPACITY, MAX_BLOCKS = 1 << 16, 1 << 30, 1 << 31  # of a page's tokens, a sequence's, all heads' blocks
MAX_VOCAB = 1 << 20


@functools.cache
def _op(name: str):
    """The operator pnfx::name (importing ops loads the library, which CPU tensors do without)."""
    from . import ops  # noqa: F401

    return getattr(torch.ops.pnfx, name).default


def _no_gradient(what: str, *tensors: torch.Tensor | None) -> None:
    """Of CPU tensors; the operators refuse for themselves."""
    for t in tensors:
        if t is not None and (torch.is_grad_enabled() and t.requires_grad or forward_ad.unpack_dual(t).tangent is not None):
            raise RuntimeError(f"{what} has no gradients: call it under torch.no_grad(), without tangents")


def _int32(x: torch.Tensor) -> torch.Tensor:
    """Whole numbers in 32 bits: those beyond become the first or last of them, which no sequence or row has either."""
    if x.dtype == torch.int32:
        return x
    return x.to(torch.int64).clamp(-(1 << 31), (1 << 31) - 1).to(torch.int32)


def _each(what: str, x: int | torch.Tensor | None, batch: int) -> tuple[torch.Tensor | None, int]:
    """A whole number for each sequence: an int32 tensor [batch], or one for all."""
    if x is None:
        return None, 0
    if not torch.is_tensor(x):
        x = operator.index(x)  # TypeError of what is no whole number
        if x < 0 or x >= 1 << 31:
            raise ValueError(f"{what} {x}")
        return None, x
    if x.is_floating_point() or x.dtype == torch.bool:
        raise TypeError(f"{what} is {x.dtype}: whole numbers")
    if x.shape != (batch,):
        raise ValueError(f"{what} has shape {tuple(x.shape)} for {batch} sequences")
    return _int32(x), 0


def whole_numbers(what: str, x: torch.Tensor | None, batch: int) -> torch.Tensor | None:
    """x as int32 [batch]: a tensor of one whole number for each sequence, or none."""
    if x is not None and not torch.is_tensor(x):
        raise TypeError(f"{what} is {type(x).__name__}: a tensor of one whole number for each sequence")
    return _each(what, x, batch)[0]


def _check_page(page: int) -> None:
    if not BLOCK <= page <= MAX_PAGE or page & (page - 1):
        raise ValueError(f"KVCache: pages of {page} tokens: a power of two from {BLOCK} to {MAX_PAGE}")


@dataclass
class KVCache:
    """Keys and values of one attention layer in 8 bits, of ``table.shape[0]`` sequences.

    Tokens come in blocks of 16, blocks in pages of ``page`` tokens (a power of two up to 65536); row b of ``table`` (int32
    [B, n]) names the pages of sequence b in order, so that sequences of any lengths share one pool.  Layers may
    share a table, and several sequences the pages of a common beginning, as long as none of them appends there (a
    page that two sequences append to in one call holds a mixture).  A sequence's pages hold at most 2^30 tokens; all
    pages have less than 2^31 blocks of a head.  A block of one head has one scale, a power of two
    2^E, held as the byte E + 127; e4m3 times such a scale is exact in bf16.

        k        uint8 [pages, H, page, D]           D: head_dim rounded up to a multiple of 16, the rest zeros
        v        uint8 [pages, H, page / 16, D, 16]  the 16 tokens of a block side by side
        k_scale  uint8 [pages, H, page / 16]         and v_scale
        raw      [B, H, 16, head_dim]                the last 16 keys before the FIR, position p at p % 16

    The cache does not know how long its sequences are: every call says where its tokens begin, ``start``, as an int32
    tensor [B] on the device (a captured graph's calls move on as it does) or one number for all, and with ``counts``
    (int32 [B]) how many of the call's N tokens each sequence has.  A tensor's numbers are not checked on the host: a
    sequence whose tokens do not fit its pages, or begin below 0, is left as it is by ``append`` and gets NaN from
    ``cached_attention``, and so does what would see a page that the table does not name (CPU tensors: ValueError).
    """

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor
    raw: torch.Tensor
    table: torch.Tensor

    def __post_init__(self):
        if self.k.dim() != 4 or self.raw.dim() != 4 or self.table.dim() != 2:
            raise ValueError(f"KVCache: k {tuple(self.k.shape)}, raw {tuple(self.raw.shape)}, table "
                             f"{tuple(self.table.shape)}")
        pages, H, page, D = self.k.shape
        B, d = self.table.shape[0], self.raw.shape[3]
        _check_page(page)
        if not 1 <= H < 1 << 20 or B >= 1 << 24 or B * H >= 1 << 31 or B and not (pages and self.table.shape[1]):
            raise ValueError(f"KVCache: {pages} pages of {H} heads, table {tuple(self.table.shape)}")
        if self.capacity > MAX_CAPACITY or pages * H * (page // BLOCK) >= MAX_BLOCKS:
            raise ValueError(f"KVCache: {pages} pages of {page} tokens and {H} heads, {self.capacity} tokens a sequence")
        if not 1 <= d <= MAX_HEAD_DIM or D != -(-d // BLOCK) * BLOCK:
            raise ValueError(f"KVCache: head size {d} (at most {MAX_HEAD_DIM}) in rows of {D}")
        shapes = {"v": (pages, H, page // BLOCK, D, BLOCK), "k_scale": (pages, H, page // BLOCK),
                  "v_scale": (pages, H, page // BLOCK), "raw": (B, H, RAW, d)}
        for name, shape in shapes.items():
            if getattr(self, name).shape != shape:
                raise ValueError(f"KVCache: {name} has shape {tuple(getattr(self, name).shape)}, not {shape}")
        for name in ("k", "v", "k_scale", "v_scale"):
            if getattr(self, name).dtype != torch.uint8:
                raise TypeError(f"KVCache: {name} is {getattr(self, name).dtype}, not uint8")
        if self.table.dtype != torch.int32:
            raise TypeError(f"KVCache: table is {self.table.dtype}, not int32")
        for name in ("k", "v", "k_scale", "v_scale", "raw", "table"):
            t = getattr(self, name)
            if not t.is_contiguous() or t.device != self.k.device:
                raise ValueError(f"KVCache: {name} must be contiguous, on k's device")

    @classmethod
    def new(cls, batch: int, n_heads: int, head_dim: int, max_len: int, page: int = 64,
            dtype: torch.dtype = torch.bfloat16, device: torch.device | str = "cuda", pages: int | None = None,
            table: torch.Tensor | None = None) -> "KVCache":
        """An empty cache for sequences of up to max_len tokens: each with pages of its own, or with a ``table`` and a
        number of ``pages`` in all.  ``dtype``: the type of the keys that will be appended."""
        _check_page(page)
        width = -(-max_len // page)
        if table is None:
            table = torch.arange(batch * width, dtype=torch.int32, device=device).view(batch, width)
        if pages is None:
            pages = batch * width
        D = -(-head_dim // BLOCK) * BLOCK

        def byte(*shape):
            return torch.zeros(shape, dtype=torch.uint8, device=device)

        return cls(byte(pages, n_heads, page, D), byte(pages, n_heads, page // BLOCK, D, BLOCK),
                   byte(pages, n_heads, page // BLOCK), byte(pages, n_heads, page // BLOCK),
                   torch.zeros(batch, n_heads, RAW, head_dim, dtype=dtype, device=device), table)

    @property
    def capacity(self) -> int:
        """Tokens that a sequence's pages hold."""
        return self.table.shape[1] * self.k.shape[2]

    def _span(self, what: str, start, counts, N: int):
        B = self.table.shape[0]
        start, at = _each("start", start, B)
        counts = whole_numbers("counts", counts, B)
        if start is None and counts is None and at + N > self.capacity:
            raise ValueError(f"{what}: tokens {at} .. {at + N - 1} in pages for {self.capacity}")
        return start, at, counts

    def append(self, k: torch.Tensor, v: torch.Tensor, start: int | torch.Tensor,
               taps: torch.Tensor | None = None, counts: torch.Tensor | None = None) -> None:
        """Writes keys and values [B, H, N, head_dim] (any strides with unit inner one) of the tokens from ``start``
        on.  With ``taps`` (fp32 [K] or [H, K], oldest lag first, K <= 16) the keys that are kept are those behind the
        causal FIR, over this call's keys and the last ones of the calls before; it is summed in 64 bits.

        A block's scale is the smallest power of two for which its numbers stay within e4m3; where a call begins inside
        a block, the tokens before its own are rounded again if the scale has to grow.  What is not finite becomes NaN.
        Appending again from an earlier ``start`` replaces what was there; with a FIR this needs the K - 1 keys before
        it among the last 16 that were appended."""
        start, at, counts = self._span("append", start, counts, k.shape[2] if k.dim() == 4 else 0)
        if self.k.is_cuda:
            _op("cache_append")(k, v, self.k, self.v, self.k_scale, self.v_scale, self.raw, self.table, start, at, counts,
                                taps)
        else:
            _no_gradient("KVCache.append", k, v, taps)
            _append(self, k, v, at if start is None else start, taps, counts)

    def read(self, first: int | torch.Tensor, count: int,
             dtype: torch.dtype | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """Dense keys (behind the FIR) and values [B, H, count, head_dim] of positions first .. first + count - 1, of
        raw's type or ``dtype``: zeros beside the sequence's pages, NaN in pages that the table does not name.  What
        positions that nothing was appended to hold is unspecified."""
        first, at = _each("first", first, self.table.shape[0])
        dtype = self.raw.dtype if dtype is None else dtype
        if self.k.is_cuda:
            return _op("cache_read")(self.k, self.v, self.k_scale, self.v_scale, self.table, first, at, int(count),
                                     self.raw.shape[3], dtype)
        return _read(self, at if first is None else first, count, dtype)


def cached_attention(q: torch.Tensor, cache: KVCache, start: int | torch.Tensor, score_tau: torch.Tensor,
                     scale: float | None = None, gamma: float | None = 0.5, causal_mask: bool = True,
                     counts: torch.Tensor | None = None) -> torch.Tensor:
    """pn_fir_tau attention (p = 10, peak gate) of query tokens ``start`` .. start + N - 1 over the cache's keys up to
    each token's own, which is appended before; without ``causal_mask`` up to the last of the call's.

    q [B, Hq, N, head_dim], Hq a multiple of the cache's heads (query head h reads key head h // (Hq // H)); returns the
    same shape, backed by [B, N, Hq, head_dim] memory, so that merging the heads is a view.  Rows past a sequence's
    ``counts`` are zeros.  scale defaults to 1/sqrt(head_dim).

    Keys and values are what their bytes stand for, exactly; scores and sums are fp32.  bf16 queries: the weights are
    rounded to bf16 (2^-8 at most, relative) for their product with the values and normalised by the sum of the rounded
    ones; fp32 queries: 24 bits throughout.  They are normalised last: values beyond 2^117 over the number of keys may
    overflow.  On the GPU a row whose first scores are far below 1 takes its powers in their unit, down to 2^-60: keys beyond
    2^60 or scores beyond 2^67 further on may then give NaN.  Bitwise repeatable for the same arguments; a sequence's last bits may be others beside other sequences, or
    in a cache of another capacity, as all lengths go into how the keys are cut and summed."""
    if q.dim() != 4 or q.shape[3] != cache.raw.shape[3]:
        raise ValueError(f"cached_attention: q {tuple(q.shape)}, the cache's head size is {cache.raw.shape[3]}")
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    has_gamma = gamma is not None and gamma > 0.0
    start, at, counts = cache._span("cached_attention", start, counts, q.shape[2])
    if cache.k.is_cuda:
        return _op("cached_attn")(q, cache.k, cache.v, cache.k_scale, cache.v_scale, cache.table, start, at, counts,
                                  score_tau, float(scale), float(gamma) if has_gamma else 0.0, has_gamma,
                                  bool(causal_mask))
    _no_gradient("cached_attention", q, score_tau)
    return _attend(q, cache, at if start is None else start, score_tau, scale, gamma if has_gamma else None,
                   causal_mask, counts)


def sample_tokens(logits: torch.Tensor, u: torch.Tensor, temperature: float | torch.Tensor = 1.0,
                  top_k: int | torch.Tensor = 0, top_p: float | torch.Tensor = 1.0,
                  min_p: float | torch.Tensor = 0.0) -> torch.Tensor:
    """One token for each row of logits [..., V] (bf16 or fp32), int64 [...], from random numbers u (fp32 [...], in
    [0, 1)).

    Tokens have the weights exp((z - max z) / temperature) and are ordered by their logits, the lower index first among
    equals.  ``top_k`` keeps the first k (0: all), ``top_p`` the fewest first ones of these that have that share of
    their weight (1: all), ``min_p`` those whose weight is at least min_p times the largest; the first is always kept.
    The token is the first, by index, at which the running weight of the kept ones is above u times their whole weight.
    temperature 0 takes the first of the order.  Each setting is one value or a tensor [...] of one for each row.

    Minus infinity is never drawn; a row that holds a NaN, or nothing else, gets -1.  GPU: weights are taken in 64 bits
    (1.4e-13) and summed as 64-bit fixed point, the largest as 2^S with S = min(50, 62 - ceil(log2 V)): the result depends on
    no order of sums, a border is off by V 2^-(S+1) of the largest weight at most, and a token of less than half a unit is
    not drawn.  A u beside [0, 1) is taken as the nearest, NaN as 0.  V <= 2^20."""
    V = logits.shape[-1] if logits.dim() else 0
    if not logits.dim() or not 1 <= V <= MAX_VOCAB:
        raise ValueError(f"sample_tokens: logits {tuple(logits.shape)}: rows of 1 to {MAX_VOCAB}")
    if logits.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"sample_tokens: logits are {logits.dtype} (float32, bfloat16)")
    rows = logits.shape[:-1]
    if u.shape != rows or u.dtype != torch.float32:
        raise ValueError(f"sample_tokens: u is {u.dtype} {tuple(u.shape)}, not float32 {tuple(rows)}")
    settings = {"temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p}
    one = dict.fromkeys(settings, 0.0)
    each = dict.fromkeys(settings)
    for name, x in settings.items():
        if torch.is_tensor(x):
            if x.shape != rows:
                raise ValueError(f"sample_tokens: {name} has shape {tuple(x.shape)}, the rows {tuple(rows)}")
            if x.is_floating_point() == (name == "top_k"):
                raise TypeError(f"sample_tokens: {name} is {x.dtype}")
            each[name] = (_int32(x) if name == "top_k" else x.to(torch.float32)).reshape(-1)
        elif not x >= 0 or (name == "top_k" and x % 1 != 0):
            raise ValueError(f"sample_tokens: {name} {x}")
        else:
            one[name] = x
    args = (one["temperature"], int(min(one["top_k"], MAX_VOCAB)), one["top_p"], one["min_p"], each["temperature"], each["top_k"],
            each["top_p"], each["min_p"])
    z, u = logits.detach().reshape(-1, V), u.detach().reshape(-1)
    return (_op("sample_tokens") if z.is_cuda else _sample)(z, u, *args).view(rows)


# ------------------------------------------------------------------------------ CPU tensors
def _two_to(e: torch.Tensor) -> torch.Tensor:
    return (e.long() + 1023 << 52).view(torch.float64)


def _checked(cache: KVCache, what: str, x: torch.Tensor, start, counts) -> tuple[torch.Tensor, torch.Tensor]:
    """start and counts as int64 [B]; what the kernels leave alone raises here."""
    B, H, d = cache.table.shape[0], cache.raw.shape[1], cache.raw.shape[3]
    if x.dim() != 4 or x.shape[0] != B or x.shape[3] != d or x.shape[1] % H:
        raise ValueError(f"{what}: {tuple(x.shape)} for a cache of B={B} H={H} head size {d}")
    if x.device != cache.k.device:
        raise ValueError(f"{what}: a tensor on {x.device}, the cache on {cache.k.device}")
    start = torch.as_tensor(start).long().expand(B)
    n = torch.full((B,), x.shape[2]) if counts is None else counts.long().clamp(0, x.shape[2])
    if ((n > 0) & ((start < 0) | (start + n > cache.capacity))).any():
        raise ValueError(f"{what}: tokens beside the {cache.capacity} that a sequence's pages hold")
    return torch.where(n > 0, start, 0), n  # of no tokens: anywhere


def _at(cache: KVCache, pos: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Page and place in it of positions [B, n] within the capacity."""
    page = cache.k.shape[2]
    return cache.table.long().gather(1, pos // page), pos % page


def _e4m3(x: torch.Tensor) -> torch.Tensor:
    """x (64 bits, at most 448) as e4m3 bytes, ties to even; NaN for what is not finite."""
    _, e = torch.frexp(x)
    step = _two_to((e - 4).clamp(min=-9))
    x = torch.where(x.isfinite(), (x / step).round() * step, torch.nan)
    return x.float().to(torch.float8_e4m3fn).view(torch.uint8)


def _need(top: torch.Tensor) -> torch.Tensor:
    m, e = torch.frexp(top / 448)
    return torch.where(m == 0.5, e - 1, e).clamp(min=LOWEST).masked_fill(top == 0, LOWEST)


def _append(cache: KVCache, k, v, start, taps, counts) -> None:
    B, H, _, d = cache.raw.shape
    if k.shape != v.shape or k.dtype != cache.raw.dtype or v.dtype != k.dtype or k.shape[1] != H:
        raise ValueError(f"append: k {k.dtype} {tuple(k.shape)}, v {v.dtype} {tuple(v.shape)} to a cache of "
                         f"{cache.raw.dtype} {tuple(cache.raw.shape)}")
    if not k.numel():
        return
    start, n = _checked(cache, "append", k, start, counts)
    N = k.shape[2]
    x = k.double()
    if taps is not None:
        taps = taps.double().reshape(-1, taps.shape[-1])
        K = taps.shape[1]
        if K > MAX_TAPS or taps.shape[0] not in (1, H):
            raise ValueError(f"append: taps {tuple(taps.shape)}")
        old = start[:, None] + torch.arange(1 - K, 0)
        hist = cache.raw.double().gather(2, (old % RAW)[:, None, :, None].expand(B, H, -1, d))
        hist = torch.where((old >= 0)[:, None, :, None], hist, 0.0)
        x = (torch.cat([hist, x], 2).unfold(2, K, 1) * taps[:, None, None]).sum(-1)
        x = torch.where(x.abs() < 2.0 ** 128, x, x * torch.inf)  # beyond fp32: not finite
    D = cache.k.shape[3]
    for b in range(B):
        s, end = int(start[b]), int(start[b] + n[b])
        for p0 in range(s // BLOCK * BLOCK, end, BLOCK) if end > s else ():
            page, place = int(cache.table[b, p0 // cache.k.shape[2]]), p0 % cache.k.shape[2]
            if not 0 <= page < cache.k.shape[0]:
                raise ValueError(f"append: page {page} of {cache.k.shape[0]}")
            t0, t1 = max(0, s - p0), min(BLOCK, end - p0)
            blk = place // BLOCK
            kb = cache.k[page, :, place:place + BLOCK]       # [H, 16, D]
            vb = cache.v[page, :, blk].transpose(1, 2)       # [H, 16, D]
            for bytes_, scale, new in ((kb, cache.k_scale[page, :, blk], x), (vb, cache.v_scale[page, :, blk], v.double())):
                new = F.pad(new[b, :, p0 + t0 - s:p0 + t1 - s], (0, D - d))
                e = _need(torch.where(new.isfinite(), new.abs(), 0.0).amax((1, 2)))
                if t0:
                    was = scale.int().clamp(max=247) - 127
                    e = torch.maximum(e, was)
                    old = bytes_[:, :t0].contiguous().view(torch.float8_e4m3fn).double()
                    bytes_[:, :t0] = _e4m3(old * _two_to(was - e)[:, None, None])
                bytes_[:, t0:t1] = _e4m3(new / _two_to(e)[:, None, None])
                scale.copy_(e + 127)
        for i in range(max(0, int(n[b]) - RAW), int(n[b])):
            cache.raw[b, :, (s + i) % RAW] = k[b, :, i]


def _read(cache: KVCache, first, count: int, dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor]:
    if count < 0 or dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"read: {count} positions as {dtype}")
    B, H, _, d = cache.raw.shape
    pos = torch.as_tensor(first).long().expand(B)[:, None] + torch.arange(count)
    there = (pos >= 0) & (pos < cache.capacity)
    page, place = _at(cache, pos.clamp(0, cache.capacity - 1))
    named = (page >= 0) & (page < cache.k.shape[0])
    page, place = torch.where(named, page, 0)[:, None], place[:, None]
    h = torch.arange(H)[:, None]
    k = cache.k[page, h, place].view(torch.float8_e4m3fn).double()
    v = cache.v[page, h, place // BLOCK, :, place % BLOCK].view(torch.float8_e4m3fn).double()
    out = []
    for x, scale in ((k, cache.k_scale), (v, cache.v_scale)):
        x = x[..., :d] * _two_to(scale[page, h, place // BLOCK].int() - 127)[..., None]
        x = torch.where(named[:, None, :, None], x, torch.nan)
        out.append(torch.where(there[:, None, :, None], x, 0.0).to(dtype))
    return out[0], out[1]


def _attend(q, cache: KVCache, start, tau, scale, gamma, causal, counts) -> torch.Tensor:
    B, Hq, N, d = q.shape
    if tau.numel() != 1:
        raise ValueError(f"cached_attention: score_tau of shape {tuple(tau.shape)}, not one value")
    tau = tau.reshape(())
    start, n = _checked(cache, "cached_attention", q, start, counts)
    o = q.new_zeros(B, N, Hq, d).transpose(1, 2)
    if not q.numel() or not n.any():
        return o
    H, L = cache.raw.shape[1], int((start + n).max())
    k, v = (t.repeat_interleave(Hq // H, 1) for t in _read(cache, 0, L, torch.float32))
    end = start[:, None] + (torch.arange(N) + 1 if causal else n[:, None])  # [B, N]
    sees = (torch.arange(L) < end.expand(B, N)[..., None]) & (torch.arange(N) < n[:, None])[..., None]
    page = cache.table.long().gather(1, torch.arange(L).expand(B, -1) // cache.k.shape[2])
    if ((page < 0) | (page >= cache.k.shape[0]))[torch.arange(L) < (start + n)[:, None]].any():
        raise ValueError(f"cached_attention: a page beside the {cache.k.shape[0]}")
    sees = sees[:, None]
    u = torch.where(sees, F.relu(q.float() @ k.transpose(2, 3) * scale - tau.float()), 0.0)
    peak = u.amax(-1, keepdim=True)
    x = u / torch.where(peak > 0, peak, 1.0)  # the powers of what may be large or small: of at most 1
    w = ((x * x) ** 2 * x) ** 2
    w = w / (w.sum(-1, keepdim=True) + 1e-12 / peak.double() ** 10).float()
    if gamma is not None:
        w = w * torch.where(peak > 0, peak / (peak + gamma), 0.0)  # gamma may be 0 in fp32
    bad = ~v.isfinite()
    y = w @ torch.where(bad, 0.0, v)
    if bad.any():  # those count where they are seen only
        y = torch.where(sees.float().expand(B, Hq, N, L) @ bad.float() > 0, torch.nan, y)
    return o.copy_(y)


def _sample(z, u, temperature, top_k, top_p, min_p, temperature_each, top_k_each, top_p_each, min_p_each):
    if not len(z):
        return torch.empty(0, dtype=torch.int64)
    V = z.shape[1]

    def setting(one, each):
        return torch.full((len(z), 1), one, dtype=torch.float64) if each is None else each.double()[:, None]

    T, k = setting(temperature, temperature_each), setting(top_k, top_k_each)
    p, least = setting(top_p, top_p_each), setting(min_p, min_p_each).clamp(max=1)
    k = torch.where(T > 0, torch.where(k <= 0, V, k), 1)
    top = z.double().amax(1, keepdim=True)
    y = torch.where(z == top, 0.0, (z.double() - top) / torch.where(T > 0, T, 1.0))
    w = torch.exp(y)
    w, order = torch.nan_to_num(w).gather(1, (by := z.sort(dim=1, descending=True, stable=True).indices)), by
    w = torch.where(torch.arange(V) < k, w, 0.0)
    before = w.cumsum(1) - w
    keep = ~(w < least) & (~(p < 1) | (before < p * w.sum(1, keepdim=True)))  # a NaN cuts nothing off
    keep[:, 0] = True
    c = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0.0)).cumsum(1)
    at = torch.nan_to_num(u.double(), nan=0.0).clamp(0, 1)[:, None] * c[:, -1:]
    last = (c < c[:, -1:]).sum(1)  # the last one that is kept: u may be 1, rounded from more bits
    token = (c <= at).sum(1).minimum(last)
    lost = z.isnan().any(1) | (z == -torch.inf).all(1)
    return torch.where(lost, -1, token)
