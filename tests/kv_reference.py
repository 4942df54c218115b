"""The attention memory's definitions in numpy: the cache's format in float32, step by
step, everything computed from it in float64."""

from __future__ import annotations

import numpy as np

Z = {"int8": np.float32(127), "fp8": np.float32(448)}
TINY = np.float32(2.0 ** -100)


def _e4m3_numbers():
    """Every finite e4m3 number that is not negative, ascending: 8 subnormals, then
    4-bit exponents 1..15 with 3-bit fractions, without the code of NaN."""
    out = [m * 2.0 ** -9 for m in range(8)]
    for e in range(1, 16):
        out += [(8 + m) * 2.0 ** (e - 10) for m in range(8)]
    return np.array(out[:-1])


E4M3 = _e4m3_numbers()


def to_e4m3(x):
    """Nearest e4m3 number of |x| <= 448, ties to the even code."""
    a = np.abs(np.asarray(x, np.float64))
    hi = np.clip(np.searchsorted(E4M3, a), 1, len(E4M3) - 1)
    lo = hi - 1
    dl, dh = a - E4M3[lo], E4M3[hi] - a
    pick = np.where(dl < dh, lo, np.where(dh < dl, hi, np.where(lo % 2 == 0, lo, hi)))
    return np.copysign(E4M3[pick], x)


def encode(y, code):
    y = np.clip(np.asarray(y, np.float32), -Z[code], Z[code])
    return np.rint(y).astype(np.float64) if code == "int8" else to_e4m3(y)


class Store:
    """Keys or values of one sequence: codes [n, h, d] (float64) and scales [blocks, h]."""

    def __init__(self, heads, dim, block, code):
        self.block, self.code = block, code
        self.codes = np.zeros((0, heads, dim))
        self.scales = np.zeros((0, heads), np.float32)

    def append(self, x):
        x = np.asarray(x, np.float32)
        at = 0
        while at < len(x):
            n = len(self.codes)
            held = n % self.block
            part = x[at:at + self.block - held]
            with np.errstate(invalid="ignore"):
                big = np.abs(part).max(axis=(0, 2))
                s = np.where(big >= TINY, big * (np.float32(1) / Z[self.code]), np.float32(0)).astype(np.float32)
                bad = ~np.isfinite(part).all(axis=(0, 2))
                if held:
                    old = self.scales[-1]
                    s = np.where(s > old, s, old)
                    bad |= np.isnan(old)
                s = np.where(bad, np.float32(np.nan), s).astype(np.float32)
                if held:
                    ratio = np.where(s > 0, old / np.where(s > 0, s, 1), 0).astype(np.float32)
                    tail = self.codes[n - held:].astype(np.float32)
                    moved = encode(np.nan_to_num(tail * ratio[None, :, None]), self.code)
                    grown = (s > old)[None, :, None]
                    self.codes[n - held:] = np.where(grown, moved, tail)
                    self.scales[-1] = s
                else:
                    self.scales = np.concatenate([self.scales, s[None]])
                inv = np.where(s > 0, np.float32(1) / np.where(s > 0, s, 1), 0).astype(np.float32)
                c = encode(np.nan_to_num(part * inv[None, :, None]), self.code)
            self.codes = np.concatenate([self.codes, c])
            at += len(part)

    def values32(self):
        s = np.repeat(self.scales, self.block, axis=0)[:len(self.codes)]
        return self.codes.astype(np.float32) * s[:, :, None]

    def values(self):
        s = np.repeat(self.scales, self.block, axis=0)[:len(self.codes)]
        return self.codes * s[:, :, None].astype(np.float64)

    def kept(self, slots):
        """The store of the slots [m, h] of each head, in blocks anew."""
        new = Store(self.codes.shape[1], self.codes.shape[2], self.block, self.code)
        heads = np.arange(self.codes.shape[1])[None]
        s = self.scales[slots // self.block, heads]
        c = self.codes[slots, heads]
        for j in range(0, len(slots), self.block):
            part = s[j:j + self.block]
            top = part.max(axis=0)  # NaN above all
            with np.errstate(invalid="ignore"):
                r = np.where(top > 0, part / np.where(top > 0, top, 1), 0).astype(np.float32)
                moved = encode(np.nan_to_num(c[j:j + self.block].astype(np.float32) * r[:, :, None]),
                               self.code)
            new.codes = np.concatenate([new.codes, moved])
            new.scales = np.concatenate([new.scales, top[None].astype(np.float32)])
        return new


def visible(n, count, causal, window):
    """[count, n]: which slots token i of the last `count` sees."""
    p = n - count + np.arange(count)[:, None]
    j = np.arange(n)[None]
    see = (j <= p) if causal else np.ones((count, n), bool)
    return see & (j > p - window) if window else see


def attend(q, k, v, see, scale):
    """q [t, hq, d], k, v [n, h, d], see [t, n]: out, lse, weights [n, h], in float64."""
    t, hq, d = q.shape
    h = k.shape[1]
    g = hq // h
    out, lse = np.zeros((t, hq, d)), np.full((t, hq), -np.inf)
    w = np.zeros((k.shape[0], h))
    rows = see.any(axis=1)
    if not rows.any():
        return out, lse, w
    q = q[rows].astype(np.float64)
    hide = ~see[rows]
    for a in range(h):
        # slots that no row sees may hold NaN: they take no part
        used = see[rows].any(axis=0)
        ka, va = k[used, a], v[used, a]
        for b in range(a * g, a * g + g):
            s = q[:, b] @ ka.T * scale
            s[hide[:, used]] = -np.inf
            m = s.max(axis=1, keepdims=True)
            with np.errstate(invalid="ignore"):
                e = np.exp(s - m)
                total = e.sum(axis=1, keepdims=True)
                p = e / total
            out[rows, b] = p @ va
            lse[rows, b] = (m + np.log(total))[:, 0]
            w[used, a] += p.sum(axis=0)
    return out, lse, w


def keep_slots(w, budget, recent):
    """Slots that stay [m, h] ascending, and those that leave: w [n, h]."""
    n, h = w.shape
    if n <= budget:
        return np.tile(np.arange(n)[:, None], (1, h)), np.zeros((0, h), int)
    stay, gone = [], []
    for a in range(h):
        key = np.where(np.isnan(w[:n - recent, a]), np.inf, w[:n - recent, a])
        nan = np.isnan(w[:n - recent, a])
        order = sorted(range(n - recent), key=lambda j: (not nan[j], -key[j], j))
        keep = sorted(order[:budget - recent]) + list(range(n - recent, n))
        stay.append(keep)
        gone.append(sorted(set(range(n)) - set(keep)))
    return np.array(stay, int).reshape(h, -1).T, np.array(gone, int).reshape(h, -1).T
