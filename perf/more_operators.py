"""The 8-bit key and value cache, attention over it and the draw of the next token: the calls whose time is measured.

Kinds of case:

* ``write``   new keys and values of each sequence go into its cache, the keys behind the causal FIR, both rounded
              to 8 bits; then the blocks that the call may have changed are read back;
* ``read``    a whole cache is read back as dense keys and values;
* ``attend``  pn_fir_tau attention (p = 10, peak gate) of the last tokens of each sequence over its cache;
* ``sample``  one token per row of logits, by temperature, top-k, top-p and min-p, from given random numbers.

The cache.  Tokens come in blocks of 16, blocks in pages, and ``table [B, n]`` names the pages of each sequence in
order.  A block of one head has one scale, a power of two 2^E, held as the byte E + 127, and its numbers over the
scale are rounded to e4m3, ties to even; what is not finite is a NaN there.

    k        [pages, H, page, D]          bytes; D is the head size rounded up to a multiple of 16, the rest zeros
    v        [pages, H, page / 16, D, 16] bytes, the 16 tokens of a block side by side
    k_scale  [pages, H, page / 16]        bytes, and v_scale
    raw      [B, H, 16, d]                the last 16 keys before the FIR, position p at p % 16

E is the smallest of -100, -99, ... for which no finite |number| is above 448 * 2^E.  A call that begins inside a block
keeps the tokens before its own: the scale is then the larger of the block's and that of the new numbers, and the kept
ones are rounded again to it.

The draw.  w_i = exp((z_i - max z) / temperature); tokens are ordered by z, the lower index first among equals.  top_k
keeps the first k, top_p the fewest first ones of these that have its share of their weight, min_p those whose weight
is at least min_p times the largest.  The token is the first, by index, at which the running weight of the kept ones
is above u times their whole weight.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
TAPS = 7
BLOCK = 16
LOWEST = -100  # smallest scale: 2^LOWEST


def _write(name, B, H, d, N, past, ragged=True, dtype="bf16", page=64):
    return dict(name=name, kind="write", B=B, H=H, d=d, N=N, past=past, ragged=ragged, dtype=dtype, page=page)


def _read(name, B, H, d, N, dtype="bf16", page=64):
    return dict(name=name, kind="read", B=B, H=H, d=d, N=N, dtype=dtype, page=page)


def _attend(name, B, Hq, H, d, N, past, ragged=True, dtype="bf16", page=64):
    return dict(name=name, kind="attend", B=B, Hq=Hq, H=H, d=d, N=N, past=past, ragged=ragged, dtype=dtype,
                page=page)


def _sample(name, B, V, temperature, top_k=0, top_p=1.0, min_p=0.0, each=False, dtype="bf16"):
    return dict(name=name, kind="sample", B=B, V=V, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p,
                each=each, dtype=dtype)


def listed():
    return [
        # Serving a batch, one layer's new token of each of 64 sequences: small, the launch counts.
        _write("write_token", 64, 16, 64, 1, 8192),
        # Prompts of 8192 tokens written into empty caches, the benchmark's long attention shape.
        _write("write_prompt", 4, 16, 64, 8192, 0, ragged=False),
        # Pieces of prompts of different lengths behind different contexts, head size and length that fit no block.
        _write("write_ragged", 7, 3, 40, 77, 1000, dtype="f32", page=16),
        # The same long prompts' cache read back whole, as for attention over dense keys.
        _read("read_back", 4, 16, 64, 8192),
        # The benchmark's language model (d_model 256, 4 heads) at the end of its 512 tokens, one sequence.
        _attend("attend_one", 1, 4, 4, 64, 1, 511, ragged=False),
        # Serving a batch: one token of each of 64 sequences behind up to 8192 others.
        _attend("attend_batch", 64, 16, 16, 64, 1, 8191),
        # Two very long contexts, key heads shared by four query heads: the largest call.
        _attend("attend_long", 2, 32, 8, 128, 1, 131071, ragged=False),
        # A prompt taken in pieces: 512 tokens behind up to 7680.
        _attend("attend_chunk", 4, 16, 16, 64, 512, 7680),
        # Full precision, three tokens checked at once, shared heads, sizes that fit no block, small pages.
        _attend("attend_f32", 5, 6, 3, 80, 3, 3001, dtype="f32", page=16),
        # The benchmark's vocabulary, one sequence.
        _sample("sample_one", 1, 33278, 0.8, top_k=50),
        # A large vocabulary and a batch whose requests have settings of their own.
        _sample("sample_batch", 256, 131072, 0.9, top_p=0.95, min_p=0.01, each=True),
        # Temperature alone, so that the whole row counts; sizes that fit no tile.
        _sample("sample_f32", 61, 50257, 1.1, dtype="f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = "f32" if rng.random() < 0.25 else "bf16"
    kind = rng.choice(["write", "read", "attend", "attend", "attend", "sample", "sample"])
    if kind == "sample":
        B, V = _log(rng, 1, 256), _log(rng, 100, 200000)
        return dict(kind=kind, B=B, V=V, temperature=rng.choice([0.6, 0.8, 1.0, 1.3]),
                    top_k=rng.choice([0, 0, 1, 20, 64, _log(rng, 2, V)]), top_p=rng.choice([1.0, 1.0, 0.5, 0.9, 0.99]),
                    min_p=rng.choice([0.0, 0.0, 0.02, 0.1]), each=rng.random() < 0.4, dtype=dtype)
    H, page = rng.choice([1, 2, 3, 4, 5, 8, 12, 16]), rng.choice([16, 32, 64, 64, 128])
    d = rng.choice([16, 32, 64, 64, 128, 128, 256, 40, 72, 80, 96, 112, rng.randint(8, 128)])
    case = dict(kind=kind, B=_log(rng, 1, 128), H=H, d=d, N=_log(rng, 1, 8192) if rng.random() < 0.6 else 1, dtype=dtype, page=page)
    if kind == "read":
        case["N"] = _log(rng, 1, 16384)
    else:
        case["past"] = rng.choice([0, _log(rng, 1, 8192), _log(rng, 64, 131072)])
        case["ragged"] = rng.random() < 0.7
    if kind == "attend":
        case["Hq"] = H * rng.choice([1, 1, 2, 4, 8])
        case["N"] = rng.choice([1, 1, 1, rng.randint(2, 8), _log(rng, 9, 1024)])
    most = 5e8  # bytes, or a fiftieth of the operations: no more than the largest listed case has

    def cost():
        w = work(case)
        return max(w["bytes"], w["flops"] / 50)

    while case["B"] > 1 and cost() > most:
        case["B"] //= 2
    while case["N"] > 1 and cost() > most:
        case["N"] //= 2
    while case.get("past", 0) > 64 and cost() > most:
        case["past"] //= 2
    return case


def _numbers(case):
    """The sizes of a cache's case: D, pages a sequence."""
    N = case["N"] + case.get("past", 0)
    return -(-case["d"] // BLOCK) * BLOCK, -(-N // case["page"])


def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    B = case["B"]
    if case["kind"] == "sample":  # the logits, the random numbers; the tokens
        return {"bytes": float(es * B * case["V"] + 12 * B), "flops": 4.0 * B * case["V"]}
    H, d, N = case["H"], case["d"], case["N"]
    one = 2 * d + 2 / BLOCK  # bytes of a token and head
    if case["kind"] == "read":  # the cache; keys and values
        return {"bytes": B * H * N * (one + 2 * es * d), "flops": 2.0 * B * H * N * d}
    if case["kind"] == "write":  # new keys and values; the cache, and what is read back of it
        back = _window(case)
        return {"bytes": B * H * (N * (2 * es * d + one) + back * (one + 2 * es * d)),
                "flops": B * H * d * (N * (2.0 * TAPS + 2) + 2 * back)}
    mean = case["past"] / (2 if case["ragged"] else 1) + N  # keys of a sequence
    pairs = B * case["Hq"] * N * (mean - (N - 1) / 2)
    return {"bytes": B * H * mean * one + 2 * es * B * case["Hq"] * N * d, "flops": 4.0 * pairs * d}


def _window(case):
    """Tokens of the blocks that a call may change."""
    behind = BLOCK - 1 if case["past"] else 0
    return -(-(case["N"] + behind) // BLOCK) * BLOCK


def _lengths(case, g):
    """Tokens that each sequence has before the call."""
    B, past = case["B"], case["past"]
    if not case["ragged"]:
        return torch.full((B,), past, dtype=torch.int32, device="cuda")
    return (torch.rand(B, generator=g, device="cuda", dtype=torch.float64) * (past + 1)).int()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    B = case["B"]

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dt)

    s = dict(case)
    if case["kind"] == "sample":
        V = case["V"]
        # a few likely tokens and a long tail: about rank^-1.3
        s["logits"] = (torch.randn(B, V, generator=g, device="cuda") * 1.5 -
                       1.3 * torch.log1p(V * torch.rand(B, V, generator=g, device="cuda"))).to(dt)
        s["u"] = torch.rand(B, generator=g, device="cuda")
        if case["each"]:  # requests' own settings, around the case's
            r = torch.rand(4, B, generator=g, device="cuda")
            s["temperature"] = case["temperature"] * (0.75 + r[0] / 2)
            s["top_k"] = (case["top_k"] * (0.5 + r[1])).int()
            s["top_p"] = torch.where(r[2] < 0.25, torch.ones_like(r[2]), case["top_p"] * (0.9 + r[2] / 10))
            s["min_p"] = case["min_p"] * 2 * r[3]
        return s

    H, d, N, page = case["H"], case["d"], case["N"], case["page"]
    D, n = _numbers(case)
    past = _lengths(case, g) if case["kind"] != "read" else None
    # what lies in the cache: numbers of about unit size, the head's own columns
    def held(*shape, columns):
        x = (torch.randn(*shape, generator=g, device="cuda") * 128).clamp_(-448, 448)
        x = x * (columns < d)
        return x.to(torch.float8_e4m3fn).view(torch.uint8)

    at = torch.arange(D, device="cuda")
    s["k"] = held(B * n, H, page, D, columns=at)
    s["v"] = held(B * n, H, page // BLOCK, D, BLOCK, columns=at[:, None])
    for name in ("k_scale", "v_scale"):
        s[name] = torch.randint(119, 122, (B * n, H, page // BLOCK), generator=g, device="cuda", dtype=torch.uint8)
    s["table"] = torch.randperm(B * n, generator=g, device="cuda").view(B, n).int()
    s["raw"] = normal(B, H, 16, d)
    s["start"] = past
    if case["kind"] == "write":
        rows = normal(B, N, 3 * H * d)  # a projection's rows: queries, keys, values
        _, s["new_k"], s["new_v"] = (t.view(B, N, H, d).transpose(1, 2) for t in rows.split(H * d, 2))
        lag = torch.arange(TAPS - 1, -1, -1, device="cuda", dtype=torch.float32)
        taps = torch.exp(-0.5 * (lag / (max(TAPS - 1, 1) / 3)) ** 2)
        s["taps"] = taps / taps.sum()
        s["first"] = past // BLOCK * BLOCK  # the blocks that the call may change
    if case["kind"] == "attend":
        s["q"] = normal(B, N, case["Hq"], d).transpose(1, 2)
        s["tau"] = torch.tensor(0.1, device="cuda")
    if own:  # the handle that a program keeps, around these buffers
        from paper_01_anti_decoy_pnfirtau_amd import KVCache

        s["cache"] = KVCache(s["k"], s["v"], s["k_scale"], s["v_scale"], s["raw"], s["table"])
    return s


# ------------------------------------------------------------------------------- plain forms
def _need(top):
    """The exponent of the smallest scale for numbers up to `top`."""
    m, e = torch.frexp(top.double() / 448)  # top / 448 = m 2^e, m in [1/2, 1)
    return torch.where(m == 0.5, e - 1, e).clamp(min=LOWEST).masked_fill(top == 0, LOWEST)


def _e4m3(x):
    """x (64 bits) rounded to e4m3, NaN where it is not finite."""
    _, e = torch.frexp(x)
    step = _two_to((e - 4).clamp(min=-9))  # four significant bits, 2^-9 below 2^-6
    return torch.where(x.isfinite(), (x / step).round() * step, torch.nan)


def _byte(x):
    return x.float().to(torch.float8_e4m3fn).view(torch.uint8)


def _held(b):
    return b.view(torch.float8_e4m3fn).float()


def _two_to(e):
    """2^e in 64 bits: the number whose exponent field is e + 1023."""
    return (e.long() + 1023 << 52).view(torch.float64)


def _places(s, pos):
    """Page and place in it of positions [B, n]; both exist for what the cases ask."""
    page = s["page"]
    pos = pos.clamp(0, s["table"].shape[1] * page - 1).long()
    return s["table"].gather(1, pos // page).long(), pos % page


def _plain_write(s):
    B, H, d, N = s["B"], s["H"], s["d"], s["N"]
    D = s["k"].shape[3]
    start = s["start"].long()
    k, v = (s[n].double() for n in ("new_k", "new_v"))
    # the FIR, over the keys before the call and its own
    old = start[:, None] - TAPS + 1 + torch.arange(TAPS - 1, device=k.device)
    hist = s["raw"].double().gather(2, (old % 16)[:, None, :, None].expand(B, H, -1, d))
    hist = hist * (old >= 0)[:, None, :, None]
    k = (torch.cat([hist, k], 2).unfold(2, TAPS, 1) * s["taps"].double()).sum(-1)
    # whole blocks: from the first that is touched to the last
    lead = start % BLOCK
    n = -(-(N + (BLOCK - 1 if s["past"] else 0)) // BLOCK)
    at = torch.arange(n * BLOCK, device=k.device) - lead[:, None]  # the token of the call at each place
    pos = at + start[:, None]
    mine, kept = (at >= 0) & (at < N), at < 0
    page, place = _places(s, pos)
    bpage, bplace = page[:, ::BLOCK], place[:, ::BLOCK] // BLOCK  # [B, n]
    live = mine.view(B, n, BLOCK).any(2)
    head = torch.arange(H, device=k.device)[:, None]
    out = []
    for name, new in (("k", k), ("v", v)):
        x = new.gather(2, at.clamp(0, N - 1)[:, None, :, None].expand(B, H, -1, d))
        x = torch.nn.functional.pad(x, (0, D - d)).view(B, H, n, BLOCK, D)
        m = mine.view(B, 1, n, BLOCK, 1)
        scale = s[name + "_scale"]
        idx = (bpage[:, None], head[None], bplace[:, None])  # [B, H, n]
        if name == "k":
            whole = s["k"].view(-1, H, s["page"] // BLOCK, BLOCK, D)
            bytes_ = whole[idx]
        else:
            whole = s["v"]
            bytes_ = whole[idx].transpose(-1, -2)
        was = scale[idx].int() - 127
        top = torch.where(m & x.isfinite(), x.abs(), 0.0).amax((3, 4))
        begun = kept.view(B, 1, n, BLOCK).any(3)
        e = torch.where(begun, torch.maximum(was, _need(top)), _need(top))
        fresh = _e4m3(x / _two_to(e)[..., None, None])
        again = _e4m3(_held(bytes_).double() * _two_to(was - e)[..., None, None])
        value = torch.where(m, _byte(fresh), torch.where(kept.view(B, 1, n, BLOCK, 1), _byte(again), bytes_))
        ok = live[:, None].expand(B, H, n)
        sel = tuple(t.expand(B, H, n)[ok] for t in idx)
        whole[sel] = value[ok] if name == "k" else value.transpose(-1, -2)[ok]
        scale[sel] = (e + 127).to(torch.uint8)[ok]
    last = torch.arange(max(0, N - 16), N, device=k.device)
    to = ((start[:, None] + last) % 16)[:, None, :, None].expand(B, H, -1, d)
    s["raw"].scatter_(2, to, s["new_k"][:, :, max(0, N - 16):])
    return [*_plain_read(s, s["first"], n * BLOCK), s["raw"]]


def _dense(s, pos):
    """Keys and values of positions [B, n] in fp32: [B, H, n, d]."""
    H, d = s["H"], s["d"]
    page, place = (t[:, None] for t in _places(s, pos))
    head = torch.arange(H, device=page.device)[None, :, None]
    k = _held(s["k"][page, head, place][..., :d])
    v = _held(s["v"].permute(0, 1, 2, 4, 3)[page, head, place // BLOCK, place % BLOCK][..., :d])
    two = [_two_to(s[n][page, head, place // BLOCK].int() - 127).float()[..., None] for n in ("k_scale", "v_scale")]
    return k * two[0], v * two[1]


def _plain_read(s, first, count):
    pos = torch.arange(count, device=s["k"].device) + (0 if first is None else first.long()[:, None])
    pos = pos.expand(s["B"], -1)
    there = ((pos >= 0) & (pos < s["table"].shape[1] * s["page"]))[:, None, :, None]
    return [torch.where(there, t, 0.0).to(DTYPES[s["dtype"]]) for t in _dense(s, pos)]


def _plain_attend(s):
    B, Hq, H, d, N = s["B"], s["Hq"], s["H"], s["d"], s["N"]
    G = Hq // H
    L = N + s["past"]
    pos = torch.arange(L, device=s["q"].device)
    k, v = _dense(s, pos.expand(B, -1))
    q = s["q"].float().reshape(B, H, G * N, d)
    u = (q @ k.transpose(2, 3)).view(B, H, G, N, L) * d ** -0.5 - s["tau"]
    sees = pos <= (s["start"].long()[:, None] + torch.arange(N, device=pos.device))[..., None]  # [B, N, L]
    u = torch.where(sees[:, None, None], u.clamp(min=0), 0.0)
    peak = u.amax(-1, keepdim=True)
    w = ((u * u) ** 2 * u) ** 2
    w = w / (w.sum(-1, keepdim=True) + 1e-12) * (peak / (peak + 0.5))
    return (w.view(B, H, G * N, L) @ v).view(B, Hq, N, d).to(DTYPES[s["dtype"]])


def _column(x, like):
    return x.to(like.dtype)[:, None] if torch.is_tensor(x) else torch.full_like(like[:, :1], x)


def _plain_sample(s):
    z, u = s["logits"].double(), s["u"].double()[:, None]
    V = s["V"]
    z, order = z.sort(dim=1, descending=True, stable=True)
    w = torch.exp((z - z[:, :1]) / _column(s["temperature"], z))
    rank = torch.arange(V, device=z.device)
    k = _column(s["top_k"], z)
    w = torch.where((k <= 0) | (rank < k), w, 0.0)
    p = _column(s["top_p"], z)
    before = w.cumsum(1) - w
    keep = (w >= _column(s["min_p"], z)) & ((p >= 1) | (before < p * w.sum(1, keepdim=True)))
    w = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0.0))
    c = w.cumsum(1)
    return (c <= u * c[:, -1:]).sum(1).clamp(max=V - 1)


# ------------------------------------------------------------------------- the framework's calls
def _own(s):
    from paper_01_anti_decoy_pnfirtau_amd import cached_attention, sample_tokens

    if s["kind"] == "sample":
        return sample_tokens(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                             min_p=s["min_p"])
    cache = s["cache"]
    if s["kind"] == "attend":
        return cached_attention(s["q"], cache, s["start"], s["tau"])
    if s["kind"] == "read":
        return list(cache.read(0, s["N"], dtype=DTYPES[s["dtype"]]))
    cache.append(s["new_k"], s["new_v"], s["start"], taps=s["taps"])
    return [*cache.read(s["first"], _window(s), dtype=DTYPES[s["dtype"]]), cache.raw]


def run(state):
    if own:
        return _own(state)
    if state["kind"] == "sample":
        return _plain_sample(state)
    if state["kind"] == "attend":
        return _plain_attend(state)
    return _plain_write(state) if state["kind"] == "write" else _plain_read(state, None, state["N"])


# ------------------------------------------------------------------------------- in 64 bits
def _grid():
    """The finite e4m3 numbers from zero up, from the format's definition: byte i stands for the i-th."""
    return torch.tensor([m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
                         for e in range(16) for m in range(8)][:127], device="cuda", dtype=torch.float64)


def _value(b):
    """What bytes stand for, before their scale."""
    i = (b & 127).long()
    x = torch.cat([_grid(), torch.tensor([math.nan], device="cuda", dtype=torch.float64)])[i]
    return torch.where(b >= 128, -x, x)


def _nearest(x):
    """The e4m3 number nearest to x, the one of even byte at ties."""
    grid = _grid()
    a = x.abs()
    hi = torch.searchsorted(grid, a.contiguous()).clamp(1, 126)
    lo = hi - 1
    up, down = grid[hi] - a, a - grid[lo]
    i = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    return torch.where(a.isfinite(), torch.copysign(grid[i], x), math.nan)


def _power(e):
    """2^e for whole e: from a table of halvings and doublings, which are exact."""
    table = torch.tensor([2.0 ** i for i in range(-400, 401)], device="cuda", dtype=torch.float64)
    return table[(e + 400).long()]


def _exact_sequence(s, b, first, last):
    """Keys and values of positions first .. last - 1 of sequence b, [H, n, d] each."""
    H, d, page = s["H"], s["d"], s["page"]
    pages = s["table"][b, first // page:-(-last // page)].long()
    skip = first // page * page

    def scaled(x, name):
        e = s[name][pages].double() - 127
        return x * _power(e).repeat_interleave(BLOCK, 2)[..., None]

    k = scaled(_value(s["k"][pages]), "k_scale")
    v = scaled(_value(s["v"][pages]).transpose(3, 4).reshape(len(pages), H, page, -1), "v_scale")
    return [t.transpose(0, 1).reshape(H, -1, t.shape[-1])[:, first - skip:last - skip, :d] for t in (k, v)]


def _exact_sample(s):
    got = []
    per = {n: s[n].tolist() if torch.is_tensor(s[n]) else [s[n]] * s["B"]
           for n in ("temperature", "top_k", "top_p", "min_p", "u")}
    for b in range(s["B"]):
        z = s["logits"][b].double()
        T, k, top_p, min_p, u = (per[n][b] for n in ("temperature", "top_k", "top_p", "min_p", "u"))
        order = torch.argsort(-z, stable=True)
        order = order[:k] if 0 < k < len(order) else order
        w = ((z[order] - z.max()) / T).exp()
        n = len(w)
        if top_p < 1:
            n = int(torch.searchsorted(w.cumsum(0), top_p * w.sum())) + 1
        kept = order[:n][w[:n] >= min_p].sort().values
        c = ((z[kept] - z.max()) / T).exp().cumsum(0)
        got.append(kept[torch.searchsorted(c, u * c[-1], right=True).clamp(max=len(kept) - 1)])
    return torch.stack(got)


def exact(case, seed):
    s = prepare(case, seed)
    B, dt = case["B"], torch.float64
    if case["kind"] == "sample":
        return _exact_sample(s)
    H, d, N = case["H"], case["d"], case["N"]
    if case["kind"] == "read":
        both = [_exact_sequence(s, b, 0, N) for b in range(B)]
        return [torch.stack([x[i] for x in both]) for i in (0, 1)]
    if case["kind"] == "attend":
        out = torch.zeros(B, case["Hq"], N, d, dtype=dt, device="cuda")
        for b, past in enumerate(s["start"].tolist()):
            k, v = _exact_sequence(s, b, 0, past + N)
            for h in range(case["Hq"]):
                j = h // (case["Hq"] // H)
                u = s["q"][b, h].double().matmul(k[j].mT) / math.sqrt(d) - s["tau"].double()
                u = torch.relu(u).tril(past)
                w = u ** 10
                gate = u.max(1, keepdim=True).values
                gate = gate / (gate + 0.5)
                out[b, h] = (w / (w.sum(1, keepdim=True) + 1e-12) * gate).matmul(v[j])
        return out
    # write: sequence by sequence, block by block
    n = _window(case)
    cap = s["table"].shape[1] * case["page"]
    back = [torch.zeros(B, H, n, d, dtype=dt, device="cuda") for _ in range(2)]
    raw = s["raw"].double()
    for b, past in enumerate(s["start"].tolist()):
        first = past // BLOCK * BLOCK
        last = min(first + n, cap)
        blocks = _exact_sequence(s, b, first, last)
        e0 = torch.stack([s[m][s["table"][b, first // case["page"]].long(), :, first % case["page"] // BLOCK]
                          for m in ("k_scale", "v_scale")]).double() - 127
        key = torch.zeros(H, TAPS - 1 + N, d, dtype=dt, device="cuda")
        key[:, TAPS - 1:] = s["new_k"][b].double()
        for j in range(1, TAPS):
            if past - j >= 0:
                key[:, TAPS - 1 - j] = raw[b, :, (past - j) % 16]
        k = sum(s["taps"][j].double() * key[:, j:j + N] for j in range(TAPS))
        for j in range(max(0, N - 16), N):
            raw[b, :, (past + j) % 16] = key[:, TAPS - 1 + j]
        for i, new in enumerate((k, s["new_v"][b].double())):
            x = blocks[i]
            lead = past - first
            size = torch.zeros(H, -(-(lead + N) // BLOCK) * BLOCK, d, dtype=dt, device="cuda")
            size[:, lead:lead + N] = new
            top = size.abs().view(H, -1, BLOCK * d).amax(2)
            e = torch.ceil(torch.log2(top / 448)).clamp(min=LOWEST)
            e = torch.where(top > 448 * _power(e), e + 1, e)
            e = torch.where((top <= 448 * _power(e - 1)) & (e > LOWEST), e - 1, e)
            if lead:
                e[:, 0] = torch.maximum(e[:, 0], e0[i])
                x[:, :lead] = _nearest(x[:, :lead] / _power(e[:, :1, None])) * _power(e[:, :1, None])
            two = _power(e).repeat_interleave(BLOCK, 1)[..., None]
            x[:, lead:lead + N] = (_nearest(size / two) * two)[:, lead:lead + N]
            tail = slice(lead + N, min(two.shape[1], x.shape[1]))  # behind the last token: old bytes, the block's scale now
            if tail.start < tail.stop:
                was = s[("k_scale", "v_scale")[i]]
                p = first + tail.start
                old = was[s["table"][b, p // case["page"]].long(), :, p % case["page"] // BLOCK].double() - 127
                x[:, tail] *= _power(e[:, -1] - old)[:, None, None]
            back[i][b, :, :last - first] = x
    return [*back, raw]
