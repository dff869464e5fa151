"""The 8-bit cache, attention over it and the draw of a token in 64 bits, from their definitions (numpy, loops)."""
import numpy as np

E4M3 = np.array([m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
                 for e in range(16) for m in range(8)][:127])  # byte i stands for the i-th


def nearest(x):
    """The e4m3 numbers nearest to x (|x| <= 448), the even byte's at ties; NaN for what is not finite."""
    a = np.abs(np.where(np.isfinite(x), x, 0.0))
    hi = np.clip(np.searchsorted(E4M3, a), 1, 126)
    up, down = E4M3[hi] - a, a - E4M3[hi - 1]
    i = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, hi - 1)
    return np.where(np.isfinite(x), np.copysign(E4M3[i], x), np.nan)


def need(top):
    e = -100
    while top > 448 * 2.0 ** e:
        e += 1
    return e


class Cache:
    """Numbers over their scale [B, H, capacity, d] of keys and values, the scales' exponents, all keys so far."""

    def __init__(self, B, H, d, capacity):
        self.x = {n: np.zeros((B, H, capacity, d)) for n in "kv"}
        self.e = {n: np.full((B, H, capacity // 16), -127) for n in "kv"}
        self.raw = np.zeros((B, H, capacity, d))

    def append(self, k, v, start, taps=None, counts=None):
        B, H, N, d = k.shape
        for b in range(B):
            s, n = int(start[b]), N if counts is None else int(counts[b])
            self.raw[b, :, s:s + n] = k[b, :, :n]
            for h in range(H):
                key = np.array(k[b, h, :n], dtype=np.float64)
                if taps is not None:
                    t = taps[h % len(taps)] if taps.ndim == 2 else taps
                    K = len(t)
                    key = np.zeros((n, d))
                    for i in range(n):
                        for j in range(K):
                            p = s + i - (K - 1) + j
                            if p >= 0:
                                key[i] += t[j] * self.raw[b, h, p]
                for name, new in (("k", key), ("v", v[b, h, :n])):
                    x, e = self.x[name][b, h], self.e[name][b, h]
                    for blk in range(s // 16, (s + n + 15) // 16 if n else 0):
                        p0, p1 = max(s, 16 * blk), min(s + n, 16 * blk + 16)
                        part = new[p0 - s:p1 - s]
                        fine = np.abs(part[np.isfinite(part)])
                        ne = need(fine.max() if fine.size else 0.0)
                        if p0 > 16 * blk:
                            ne = max(ne, e[blk])
                            kept = x[16 * blk:p0]
                            x[16 * blk:p0] = nearest(kept * 2.0 ** float(e[blk] - ne))
                        x[p0:p1] = nearest(part / 2.0 ** ne)
                        e[blk] = ne

    def dense(self):
        return [self.x[n] * 2.0 ** np.repeat(self.e[n], 16, 2)[..., None] for n in "kv"]


def attend(q, k, v, start, tau, scale, gamma, causal=True, counts=None, low=False, n_sum=None):
    """(O, how far fp32 sums, and weights rounded to bf16 if `low`, may be from it)."""
    B, Hq, N, d = q.shape
    G = Hq // k.shape[1]
    out, tol = np.zeros_like(q), np.zeros_like(q)
    half = 2.0 ** -24
    for b in range(B):
        n = N if counts is None else int(counts[b])
        for h in range(Hq):
            for i in range(n):
                L = int(start[b]) + (i + 1 if causal else n)
                kk, vv = k[b, h // G, :L], v[b, h // G, :L]
                s = kk @ q[b, h, i] * scale
                size = np.abs(kk) @ np.abs(q[b, h, i]) * scale
                u = np.maximum(s - tau, 0)
                # products and sum of the score, its scale and tau's subtraction
                du = half * ((d + 6) * size + 2 * np.abs(s) + 2 * abs(tau))
                P = u ** 10
                Z, M = P.sum() + 1e-12, (u.max() if L else 0.0)
                gate = 1.0 if gamma is None else M / (M + gamma)
                w = P / Z * gate
                out[b, h, i] = w @ vv
                # each power and its sums; the weights rounded twice (numerator, normaliser)
                rel = half * (12 + 3 * L) + (2 * 2.0 ** -8 if low else 0)
                dP = np.maximum((u + du) ** 10 - P, P - np.maximum(u - du, 0) ** 10)
                dw = dP / Z * gate
                dgate = 0.0 if gamma is None else 2 * (du.max() if L else 0.0) / gamma + 4 * half
                tol[b, h, i] = ((w * rel + dw) @ np.abs(vv) + (dw.sum() + dgate) * (w @ np.abs(vv))) * 1.01
    return out, tol + np.abs(out) * ((2.0 ** -8 if low else half)) + 1e-30


def sample(z, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One row's token, and how near u is to a border, as a share of the kept ones' weight."""
    z = np.asarray(z, dtype=np.float64)
    if np.isnan(z).any() or (z == -np.inf).all():
        return -1, 1.0
    order = np.lexsort((np.arange(len(z)), -z))
    if not temperature > 0:
        return int(order[0]), 1.0
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(z == z.max(), 1.0, np.exp((z - z.max()) / temperature))
    kept = order[:top_k] if 0 < top_k < len(z) else order
    if top_p < 1:
        c = np.cumsum(w[kept])
        kept = kept[:int(np.searchsorted(c, top_p * c[-1])) + 1]
    kept = np.sort(np.append(kept[1:][w[kept[1:]] >= min(min_p, 1.0)], kept[0]))
    c = np.cumsum(w[kept])
    at = u * c[-1]
    return int(kept[min(int(np.searchsorted(c, at, side="right")), len(kept) - 1)]), float(np.abs(c - at).min() / c[-1])
