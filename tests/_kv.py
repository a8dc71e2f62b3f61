"""The 8-bit key/value cache in plain 64-bit numpy: the oracle of the cache's
tests.  Everything here is a loop over tokens, heads and the layout's
definition; nothing of the library is used."""
from __future__ import annotations

import numpy as np

PAGE = 64


def padded(D: int) -> int:
    return (D + 31) // 32 * 32


def slot(t: int) -> int:
    """Byte of page token t in a value row (longhorn_hip.h)."""
    return 16 * ((t >> 2) & 3) + 8 * (t >> 5) + 4 * ((t >> 4) & 1) + (t & 3)


SLOTS = np.array([slot(t) for t in range(PAGE)])


def e4m3_values() -> np.ndarray:
    out = np.empty(256)
    for c in range(256):
        e, m = c >> 3 & 15, c & 7
        x = np.nan if e == 15 and m == 7 else m * 2.0 ** -9 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        out[c] = -x if c >> 7 else x
    return out


def code_values(fmt: str) -> np.ndarray:
    return e4m3_values() if fmt == "fp8" else np.where(np.arange(256) > 127, np.arange(256) - 256.0, np.arange(256.0))


class HostCache:
    """Codes and scales as the library's layout names them, in host memory."""

    def __init__(self, fmt, pages, H, D, seed=None):
        self.fmt, self.pages, self.H, self.D, self.Dp = fmt, pages, H, D, padded(D)
        g = np.random.default_rng(seed)
        kshape, vshape = (pages, H, PAGE, self.Dp), (pages, H, self.Dp, PAGE)
        if seed is None:
            self.k, self.v = np.zeros(kshape, np.uint8), np.zeros(vshape, np.uint8)
            self.ks, self.vs = np.zeros((pages, H, PAGE), np.float32), np.zeros((pages, H, PAGE), np.float32)
            return
        # codes of normal values; e4m3's NaN code is left out
        self.k, self.v = self._codes(g, kshape), self._codes(g, vshape)
        self.k[..., D:] = 0
        self.v[:, :, D:] = 0
        self.ks = (np.exp(0.4 * g.standard_normal((pages, H, PAGE))) * 0.01).astype(np.float32)
        self.vs = (np.exp(0.4 * g.standard_normal((pages, H, PAGE))) * 0.01).astype(np.float32)
        if fmt == "fp8":
            self.ks /= 4
            self.vs /= 4

    def _codes(self, g, shape):
        if self.fmt == "int8":
            return np.clip(np.rint(g.standard_normal(shape) * 40), -127, 127).astype(np.int8).view(np.uint8)
        c = g.integers(0, 256, shape).astype(np.uint8)
        return np.where((c & 0x7f) == 0x7f, c & 0x80, c).astype(np.uint8)

    def put(self, page, h, t, kc, vc, sk, sv):
        """One token of one head."""
        self.k[page, h, t, :self.D] = kc
        self.k[page, h, t, self.D:] = 0
        self.v[page, h, :self.D, slot(t)] = vc
        self.v[page, h, self.D:, slot(t)] = 0
        self.ks[page, h, t], self.vs[page, h, t] = sk, sv

    def token(self, page, h, t):
        """(k, v) of one token of one head in 64 bits."""
        val = code_values(self.fmt)
        with np.errstate(invalid="ignore"):
            return (val[self.k[page, h, t, :self.D]] * np.float64(self.ks[page, h, t]),
                    val[self.v[page, h, :self.D, slot(t)]] * np.float64(self.vs[page, h, t]))

    def page_values(self, page, h):
        """(k, v) [64, D] of one page and head in 64 bits."""
        val = code_values(self.fmt)
        with np.errstate(invalid="ignore"):
            k = val[self.k[page, h, :, :self.D]] * self.ks[page, h].astype(np.float64)[:, None]
            v = val[self.v[page, h, :self.D][:, SLOTS].T] * self.vs[page, h].astype(np.float64)[:, None]
        return k, v

    def find(self, table, s, pos):
        """(page, token) of a position, or None."""
        p = pos // PAGE
        if pos < 0 or p >= table.shape[1] or not 0 <= table[s, p] < self.pages:
            return None
        return int(table[s, p]), pos % PAGE

    def device(self, ops):
        """The library's handle on a copy on the GPU."""
        return ops.KvCache(self.fmt, self.pages, self.H, self.D, ops.dev(self.k), ops.dev(self.v), ops.dev(self.ks),
                           ops.dev(self.vs))


def block_table(g, lengths, pages, width=None):
    """Random distinct pages for each sequence's tokens, -1 past them."""
    need = [-(-n // PAGE) for n in lengths]
    width = max(1, max(need)) if width is None else width
    order = g.permutation(pages)
    assert sum(need) <= pages
    table, at = np.full((len(lengths), width), -1, np.int32), 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    return table


def attention(c: HostCache, q, offsets, lengths, table, k_new, v_new, tree, scale):
    """(out, bound): attention in 64 bits, and how far a kernel may be from it.

    The bound of one output, with p the softmax weights, n the tokens seen:
      2^-8 |o|                      the result's rounding to bf16
      A 2^-11                       each weight times its value scale rounded to fp16, A = sum p |v|
      A (2 ds + (n + 64) 2^-24)     fp32: scores off by ds move a weight by e^ds, and sum and
                                    products of n weights (exp2 and its argument among the 64)
      max|v| 2^-30                  fp16 subnormals of weights, queries, keys and values that are
                                    scaled so that the largest is near the top of the range
    with ds = (D + 8) 2^-24 scale max_j sum |q k_j|, an fp32 sum of D products."""
    n, Hq, D = q.shape
    G = Hq // c.H
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for s in range(len(lengths)):
        lo, hi = int(offsets[s]), int(offsets[s + 1])
        for h in range(c.H):
            ks, vs, L = [], [], max(0, int(lengths[s]))
            for p in range(-(-L // PAGE)):
                if c.find(table, s, p * PAGE) is None:
                    continue
                k, v = c.page_values(int(table[s, p]), h)
                ks.append(k[:L - p * PAGE])
                vs.append(v[:L - p * PAGE])
            cached = sum(len(k) for k in ks)
            if k_new is not None:
                ks.append(k_new[lo:hi, h].astype(np.float64))
                vs.append(v_new[lo:hi, h].astype(np.float64))
            k = np.concatenate(ks) if ks else np.zeros((0, D))
            v = np.concatenate(vs) if vs else np.zeros((0, D))
            for i in range(lo, hi):
                seen = np.ones(len(k), bool)
                if k_new is not None:
                    word = (1 << (i - lo + 1)) - 1 if tree is None else int(tree[i])
                    seen[cached:] = [(word >> j) & 1 for j in range(hi - lo)]
                if not seen.any():
                    continue
                kk, vv = k[seen], v[seen]
                for hq in range(h * G, (h + 1) * G):
                    qq = q[i, hq].astype(np.float64)
                    x = kk @ qq * scale
                    p = np.exp(x - x.max())
                    p /= p.sum()
                    out[i, hq] = p @ vv
                    ds = (D + 8) * 2.0 ** -24 * scale * (np.abs(kk) @ np.abs(qq)).max()
                    A = p @ np.abs(vv)
                    bound[i, hq] = (2.0 ** -8 * np.abs(out[i, hq])
                                    + A * (2.0 ** -11 + 2 * ds + (len(kk) + 64) * 2.0 ** -24)
                                    + np.abs(vv).max() * 2.0 ** -30)
    return out, bound
