"""Causal attention over the 8-bit cache and new tokens in 64-bit numpy, how far
a kernel may be from it, and the cases that the prefill tests run."""
from __future__ import annotations

import numpy as np

from tests import _data as D
from tests import _kv


def attention(c, q, offsets, lengths, table, k_new, v_new, scale):
    """(out, bound) of rows that sequences own; out and bound are zero elsewhere.
    c: a _kv.HostCache, or None.

    The bound of one output, with p the softmax weights, n the keys seen:
      2^-8 |o|                      the result's rounding to bf16
      A 2^-8                        each weight (times its value scale) rounded to bf16, A = sum p |v|
      A (2 ds + (n + 64) 2^-24)     fp32: scores off by ds move a weight by e^ds, and sum and
                                    products of n weights (exp2 and its argument among the 64)
      max|v| 2^-100                 weights under bf16's normal numbers
    with ds = (D + 8) 2^-24 scale max_j sum |q k_j|, an fp32 sum of D products."""
    n, Hq, dim = q.shape
    H = c.H if c is not None else k_new.shape[1]
    G = Hq // H
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for s in range(len(offsets) - 1):
        lo, hi = int(offsets[s]), int(offsets[s + 1])
        if hi <= lo:
            continue
        T, L = hi - lo, 0 if c is None else max(0, int(lengths[s]))
        for h in range(H):
            ks, vs = [np.zeros((0, dim))], [np.zeros((0, dim))]
            for p in range(-(-L // _kv.PAGE)):
                if c.find(table, s, p * _kv.PAGE) is None:
                    continue
                k, v = c.page_values(int(table[s, p]), h)
                ks.append(k[:L - p * _kv.PAGE])
                vs.append(v[:L - p * _kv.PAGE])
            cached = sum(len(k) for k in ks)
            if k_new is not None:
                ks.append(k_new[lo:hi, h].astype(np.float64))
                vs.append(v_new[lo:hi, h].astype(np.float64))
            k, v = np.concatenate(ks), np.concatenate(vs)
            if not len(k):
                continue
            seen = np.arange(len(k)) < cached + 1 + np.arange(T)[:, None]
            for hq in range(h * G, (h + 1) * G):
                qq = q[lo:hi, hq].astype(np.float64)
                with np.errstate(invalid="ignore", over="ignore"):
                    x = np.where(seen, qq @ k.T * scale, -np.inf)
                    p = np.exp(x - x.max(axis=1, keepdims=True))
                    p /= p.sum(axis=1, keepdims=True)
                    # what a row does not see is not there, whatever it holds
                    vv = np.where(np.isfinite(v), v, 0.0)
                    o = p @ vv
                    for j in np.nonzero(~np.isfinite(v).all(axis=1))[0]:
                        o = np.where(seen[:, j:j + 1] & ~np.isfinite(v[j]), o + v[j], o)
                    ds = (dim + 8) * 2.0 ** -24 * scale * np.where(seen, np.abs(qq) @ np.abs(k).T, 0).max(axis=1, keepdims=True)
                    A = p @ np.abs(vv)
                    out[lo:hi, hq] = o
                    bound[lo:hi, hq] = (2.0 ** -8 * np.abs(o) + A * (2.0 ** -8 + 2 * ds + (len(k) + 64) * 2.0 ** -24)
                                        + np.abs(vv).max() * 2.0 ** -100)
    return out, bound


class Case:
    """Packed new rows, a cache (fmt None: none) and its table."""

    def __init__(self, oracle, fmt, Hq, H, dim, lengths, new, seed, gain=1.0, spare=2, width=None, pad=0):
        g = np.random.default_rng(seed)
        self.Hq, self.H, self.dim, self.fmt = Hq, H, dim, fmt
        self.lengths, self.new = np.array(lengths, np.int32), list(new)
        n = sum(new)
        self.offs = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.scale = dim ** -0.5

        def rows(heads, by):
            return D.to_bf16_bits(oracle, (g.standard_normal((n + pad, heads, dim)) * by).astype(np.float32))
        self.q, self.k, self.v = rows(Hq, 2.0 * gain), rows(H, 1.0), rows(H, 1.0)
        self.c, self.table = None, None
        if fmt is not None:
            pages = sum(-(-int(t) // _kv.PAGE) for t in lengths) + spare
            self.c = _kv.HostCache(fmt, pages, H, dim, seed=seed + 1)
            self.table = _kv.block_table(g, [int(t) for t in lengths], pages, width)

    def want(self, new_tokens=True):
        f = D.bf16_bits_to_f32
        return attention(self.c, f(self.q), self.offs, self.lengths, self.table, f(self.k) if new_tokens else None,
                         f(self.v) if new_tokens else None, self.scale)

    def args(self, ops, wide=False, shift=0, new_tokens=True):
        """q, k, v on the GPU: apart, or slices of one row (with `shift` elements before it)."""
        if not wide:
            q, k, v = (ops.dev(x) for x in (self.q, self.k, self.v))
        else:
            import torch
            n, parts = len(self.q), [self.q.reshape(len(self.q), -1), self.k.reshape(len(self.q), -1),
                                     self.v.reshape(len(self.q), -1)]
            width = sum(p.shape[1] for p in parts)
            buf = torch.full((n * (width + shift) + shift,), 0x7fc0, dtype=torch.int16, device="cuda")
            rows = buf[shift:shift + n * (width + shift)].view(n, width + shift)[:, :width]
            rows.copy_(ops.dev(np.concatenate(parts, axis=1)))
            q, k, v = rows.split([p.shape[1] for p in parts], dim=1)
        return (q, k, v) if new_tokens else (q, None, None)

    def run(self, ops, workspace=True, wide=False, shift=0, new_tokens=True, out=None):
        q, k, v = self.args(ops, wide, shift, new_tokens)
        B = len(self.new)
        ws = ops.prefill_workspace(B, len(self.q), self.Hq, self.H, self.dim) if workspace else None
        if self.fmt is None:
            return ops.attn_prompt(q, k, v, ops.dev(self.offs), self.dim, scale=self.scale, workspace=ws, out=out)
        return ops.kv_prefill(self.c.device(ops), q, ops.dev(self.offs), ops.dev(self.lengths), ops.dev(self.table), k, v,
                              scale=self.scale, workspace=ws, out=out)


def check(got, want, bound, rows=slice(None)):
    got, want, bound = got[rows], want[rows], bound[rows]
    odd = ~np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[odd & ~np.isnan(want)], want[odd & ~np.isnan(want)])
    off = np.where(odd, 0, np.abs(got - np.where(odd, 0, want)) - bound)
    off = np.where(np.isnan(got) & odd, 0, off)
    assert (off <= 0).all(), f"{(off > 0).sum()} of {off.size} off, worst {off.max():.3g} at {np.unravel_index(off.argmax(), off.shape)}"
