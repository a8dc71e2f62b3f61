"""One attention layer of a serving step on the 8-bit key/value cache.

Prompts go in by chunks of 64 tokens: the fused int4 projection gives their
queries, keys and values, the chunk attends the cache and itself, its keys and
values are quantized into the cache.  Then every step verifies a drafted tree of
tokens for each sequence, accepts a path of it and writes the accepted tokens'
keys and values, picked out of all drafted rows.  At the end the last step is
computed again in 64 bits from what the cache reads back.

    python examples/speculative_decode.py [--fmt int8|fp8] [--steps N]
"""
from __future__ import annotations

import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from longhornai_amd import ops  # noqa: E402

HIDDEN, HEADS, KV_HEADS, DIM, GROUP = 2048, 16, 4, 128, 128
CHUNK = 64  # new tokens of a sequence that one call attends


def int4_weights(K: int, N: int, g: np.random.Generator) -> ops.W4Weights:
    """A random int4 projection whose outputs are about as large as its inputs."""
    codes = g.integers(0, 256, (K // 2, N), dtype=np.uint8)
    scales = np.full((K // GROUP, N), 1 / (4.6 * K ** 0.5), np.float16)
    zeros = np.full((K // GROUP, N), 8, np.uint8)
    return ops.prepack_w4_asym(ops.dev(codes), ops.dev(scales.view(np.uint16)), ops.dev(zeros), K, N, GROUP)


class Layer:
    """The projections, the cache and the page lists of a batch of sequences."""

    def __init__(self, fmt: str, seqs: int, most_tokens: int, seed: int):
        g = np.random.default_rng(seed)
        self.qkv = int4_weights(HIDDEN, (HEADS + 2 * KV_HEADS) * DIM, g)
        self.out = int4_weights(HEADS * DIM, HIDDEN, g)
        pages = -(-most_tokens // ops.KV_PAGE)
        self.cache = ops.kv_cache(fmt, seqs * pages, KV_HEADS, DIM)
        self.table = ops.dev(g.permutation(seqs * pages).astype(np.int32).reshape(seqs, pages))
        self.lengths = np.zeros(seqs, np.int32)
        self.workspace = {}

    def attend(self, x: torch.Tensor, new: list[int], tree: torch.Tensor | None = None):
        """New tokens' hidden states [n, HIDDEN] (bf16 bits), new[s] rows of
        sequence s, through the layer; returns (output, attention, q, k, v)."""
        wide = ops.gemm_w4a16_bf16(x, self.qkv)
        q, k, v = wide.split([HEADS * DIM, KV_HEADS * DIM, KV_HEADS * DIM], dim=1)
        offsets = ops.dev(np.concatenate([[0], np.cumsum(new)]).astype(np.int32))
        key = (len(x), max(new))
        if key not in self.workspace:
            self.workspace[key] = ops.kv_attn_workspace(self.cache, len(new), len(x), max(new), self.table.shape[1], HEADS)
        o = ops.kv_attn(self.cache, q, offsets, ops.dev(self.lengths), self.table, k, v, tree=tree, max_new=max(new),
                        workspace=self.workspace[key])
        return ops.gemm_w4a16_bf16(o.view(len(x), HEADS * DIM), self.out), o, q, k, v

    def keep(self, k: torch.Tensor, v: torch.Tensor, kept: list[int], rows: np.ndarray | None = None) -> None:
        """Writes kept[s] tokens of each sequence behind the ones it holds."""
        offsets = ops.dev(np.concatenate([[0], np.cumsum(kept)]).astype(np.int32))
        ops.kv_write(self.cache, k, v, offsets, ops.dev(self.lengths), self.table,
                     rows=None if rows is None else ops.dev(rows))
        self.lengths += np.array(kept, np.int32)


def hidden(n: int, g: torch.Generator) -> torch.Tensor:
    return torch.randn((n, HIDDEN), generator=g, device="cuda").to(torch.bfloat16).view(torch.int16)


def draft(T: int, g: np.random.Generator):
    """A tree of T tokens: (ancestor masks, a path from the root to a leaf)."""
    parents = [-1] + [int(g.integers(max(0, i - 3), i)) for i in range(1, T)]
    masks = []
    for i, p in enumerate(parents):
        masks.append((masks[p] if p >= 0 else 0) | 1 << i)
    return masks, [j for j in range(T) if masks[-1] >> j & 1]


def plain_attention(layer: Layer, s: int, q, k, v, masks) -> np.ndarray:
    """Sequence s's drafted rows attended in 64 bits over the cache as it reads back."""
    L = int(layer.lengths[s])
    ck, cv = (ops.host(t).astype(np.float64) for t in ops.kv_read(
        layer.cache, ops.dev(np.array([0, L], np.int32)), ops.dev(np.zeros(1, np.int32)), layer.table[s:s + 1], L,
        bf16=False))
    q, k, v = (t.view(torch.bfloat16).double().cpu().numpy().reshape(len(t), -1, DIM) for t in
               (x.contiguous() for x in (q, k, v)))
    out = np.zeros((len(q), HEADS, DIM))
    seen = np.array([[m >> j & 1 for j in range(len(q))] for m in masks], bool)
    seen = np.concatenate([np.ones((len(q), L), bool), seen], axis=1)
    for h in range(HEADS):
        kh = h // (HEADS // KV_HEADS)
        keys, values = np.concatenate([ck[:, kh], k[:, kh]]), np.concatenate([cv[:, kh], v[:, kh]])
        score = np.where(seen, q[:, h] @ keys.T * DIM ** -0.5, -np.inf)
        p = np.exp(score - score.max(axis=1, keepdims=True))
        out[:, h] = (p / p.sum(axis=1, keepdims=True)) @ values
    return out


def main(fmt: str = "int8", steps: int = 4, prompts: tuple[int, ...] = (300, 64, 129, 1), T: int = 12) -> float:
    """Returns the last step's largest error, relative to its largest value."""
    if steps < 1:
        raise ValueError("speculative_decode: the last step is checked, so there must be one")
    g, tg = np.random.default_rng(1), torch.Generator(device="cuda").manual_seed(1)
    layer = Layer(fmt, len(prompts), max(prompts) + steps * T, seed=2)
    left = list(prompts)
    while any(left):
        new = [min(n, CHUNK) for n in left]
        _, _, _, k, v = layer.attend(hidden(sum(new), tg), new)
        layer.keep(k, v, new)
        left = [a - b for a, b in zip(left, new)]
    worst = 0.0
    for step in range(steps):
        trees = [draft(T, g) for _ in prompts]
        words = np.array([m for masks, _ in trees for m in masks], np.int64)
        _, o, q, k, v = layer.attend(hidden(T * len(prompts), tg), [T] * len(prompts), tree=ops.dev(words))
        if step == steps - 1:
            got = o.view(torch.bfloat16).double().cpu().numpy()
            want = np.concatenate([plain_attention(layer, s, *(t[s * T:(s + 1) * T] for t in (q, k, v)), trees[s][0])
                                   for s in range(len(prompts))])
            worst = float(np.abs(got - want).max() / np.abs(want).max())
        rows = np.array([s * T + i for s, (_, path) in enumerate(trees) for i in path], np.int32)
        layer.keep(k, v, [len(path) for _, path in trees], rows)
        print(f"step {step}: accepted {[len(path) for _, path in trees]} of {T}, lengths {layer.lengths.tolist()}")
    print(f"{fmt}: the last step against 64 bits over the cache: {worst:.1e} of the largest value")
    return worst


def run(argv: list[str] | None = None) -> int:
    """The command: 0 where the last step holds to 64 bits, else 1."""
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--fmt", choices=("int8", "fp8"), default="int8")
    ap.add_argument("--steps", type=int, default=4)
    a = ap.parse_args(argv)
    if a.steps < 1:
        ap.error("--steps must be 1 or more")
    return 0 if main(a.fmt, a.steps) <= 2.0 ** -8 else 1  # (a NaN is no success)


if __name__ == "__main__":
    sys.exit(run())
