"""One attention layer of a server that batches requests as they come.

Requests with prompts of different lengths share one 8-bit cache.  Every step
takes what each running request has to give, a chunk of its prompt or one token:
the tables come from the lengths on the GPU (pages of requests that are over are
handed out again), the fused int4 projection gives queries, keys and values, the
heads are normed and turned by their positions in place, the new tokens attend the
cache and themselves, and their keys and values are quantized into it.  The last
step is computed again in 64 bits from what the cache reads back.

    python examples/serve_requests.py [--fmt int8|fp8] [--chunk N]
"""
from __future__ import annotations

import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from examples.speculative_decode import DIM, GROUP, HEADS, HIDDEN, KV_HEADS, int4_weights  # noqa: E402,F401
from longhornai_amd import ops  # noqa: E402

PAGES_A_ROW = 24  # of the block table: 1536 tokens a request


class Server:
    """The layer's weights, the cache with its free pages, and the running requests."""

    def __init__(self, fmt: str, places: int, pages: int, seed: int):
        g = np.random.default_rng(seed)
        self.qkv = int4_weights(HIDDEN, (HEADS + 2 * KV_HEADS) * DIM, g)
        self.out = int4_weights(HEADS * DIM, HIDDEN, g)
        self.turns = ops.rope_plan(DIM, theta=500000.0, scaling="yarn", factor=4.0, original=512)
        self.norms = [torch.linspace(0.5, 1.5, DIM, device="cuda").to(torch.bfloat16).view(torch.int16) for _ in range(2)]
        self.cache = ops.kv_cache(fmt, pages, KV_HEADS, DIM)
        self.table = torch.full((places, PAGES_A_ROW), -1, dtype=torch.int32, device="cuda")
        self.free = ops.dev(g.permutation(pages).astype(np.int32))
        self.left = ops.dev(np.array([pages, 0], np.int32))
        self.owned = torch.zeros(places, dtype=torch.int32, device="cuda")
        self.lengths = np.zeros(places, np.int32)  # the host's copy: it decides who gives what

    def tables(self, lengths: torch.Tensor, new: list[int]) -> ops.KvPlan:
        """The tables of a step with new[s] tokens of each place's request (-1: it is over)."""
        plan = ops.kv_plan(lengths, ops.dev(np.array(new, np.int32)), self.free, self.left, self.table,
                           sum(t for t in new if t > 0), owned=self.owned)
        self.left = plan.left
        return plan

    def step(self, x: torch.Tensor, new: list[int]):
        """Hidden states [n, HIDDEN] (bf16 bits) of the new tokens through the layer; returns
        (output, attention, q, k, v, plan)."""
        lengths = ops.dev(self.lengths)
        plan = self.tables(lengths, new)
        wide = ops.gemm_w4a16_bf16(x, self.qkv)
        q, k, v = wide.split([HEADS * DIM, KV_HEADS * DIM, KV_HEADS * DIM], dim=1)
        ops.rope(self.turns, q, k, plan.positions, q_weight=self.norms[0], k_weight=self.norms[1], out=(q, k))
        if max(new) > 1:
            ws = ops.prefill_workspace(len(new), len(x), HEADS, KV_HEADS, DIM)
            o = ops.kv_prefill(self.cache, q, plan.offsets, lengths, self.table, k, v, workspace=ws)
        else:
            ws = ops.kv_attn_workspace(self.cache, len(new), len(x), 1, PAGES_A_ROW, HEADS)
            o = ops.kv_attn(self.cache, q, plan.offsets, lengths, self.table, k, v, max_new=1, workspace=ws)
        ops.kv_write(self.cache, k, v, plan.offsets, lengths, self.table)
        return ops.gemm_w4a16_bf16(o.view(len(x), HEADS * DIM), self.out), o, q, k, v, plan

    def attended(self, s: int, L: int, q, k, v) -> np.ndarray:
        """New rows of place s after its first L tokens, attended in 64 bits over the cache as it reads back."""
        ck, cv = (ops.host(t).astype(np.float64) for t in ops.kv_read(
            self.cache, ops.dev(np.array([0, L], np.int32)), ops.dev(np.zeros(1, np.int32)), self.table[s:s + 1], L, bf16=False))
        q, k, v = (t.contiguous().view(torch.bfloat16).double().cpu().numpy().reshape(len(t), -1, DIM) for t in (q, k, v))
        T, out = len(q), np.zeros((len(q), HEADS, DIM))
        seen = np.arange(L + T) <= L + np.arange(T)[:, None]
        for h in range(HEADS):
            kh = h // (HEADS // KV_HEADS)
            keys, values = np.concatenate([ck[:, kh], k[:, kh]]), np.concatenate([cv[:, kh], v[:, kh]])
            score = np.where(seen, q[:, h] @ keys.T * DIM ** -0.5, -np.inf)
            p = np.exp(score - score.max(axis=1, keepdims=True))
            out[:, h] = (p / p.sum(axis=1, keepdims=True)) @ values
        return out


def main(fmt: str = "int8", chunk: int = 256, places: int = 3,
         requests: tuple[tuple[int, int], ...] = ((700, 3), (1, 9), (300, 4), (64, 12), (129, 5))) -> float:
    """Serves requests (prompt, tokens to make); returns the largest error of a step that holds
    both a chunk and a decoded token, and of the last step, relative to its largest value."""
    if chunk < 1:
        raise ValueError("serve_requests: a chunk has a token or more")
    tg = torch.Generator(device="cuda").manual_seed(1)
    pages = sum(-(-(p + t) // ops.KV_PAGE) for p, t in requests) - 3  # under what all of them need: some are handed out again
    server, waiting = Server(fmt, places, pages, seed=2), list(requests)
    running: list[list[int] | None] = [None] * places  # [prompt tokens left, tokens left to make]
    worst, steps, mixed = 0.0, 0, False
    while waiting or any(r is not None for r in running):
        new = []
        for s in range(places):
            if running[s] is None and waiting:
                running[s] = list(waiting.pop(0))
            r = running[s]
            new.append(0 if r is None else min(r[0], chunk) if r[0] else 1 if r[1] else -1)
        n, before = sum(t for t in new if t > 0), server.lengths.copy()
        if n:
            x = torch.randn((n, HIDDEN), generator=tg, device="cuda").to(torch.bfloat16).view(torch.int16)
            _, o, q, k, v, plan = server.step(x, new)
        else:  # (requests that are over, no other)
            plan = server.tables(ops.dev(server.lengths), new)
        last = not waiting and sum(max(r[0] + r[1], 0) for r in running if r) - n <= 0
        check = n and (last or (not mixed and max(new) > 1 and 1 in new))
        at = 0
        for s, t in enumerate(new):
            if t < 0:
                running[s], server.lengths[s] = None, 0
            elif t:
                if check:
                    rows = slice(at, at + t)
                    want = server.attended(s, int(before[s]), q[rows], k[rows], v[rows])
                    got = o[rows].view(torch.bfloat16).double().cpu().numpy()
                    worst = max(worst, float(np.abs(got - want).max() / np.abs(want).max()))
                    mixed = True
                server.lengths[s] += t
                running[s][0 if running[s][0] else 1] -= t
                at += t
        steps += 1
        left, missing = ops.host(plan.left)
        print(f"step {steps}: new tokens {new}, lengths {server.lengths.tolist()}, {left} of {pages} pages left")
        if missing:
            raise RuntimeError("serve_requests: the cache has too few pages")
    if left != pages:
        raise RuntimeError(f"serve_requests: {left} of {pages} pages came back")
    print(f"{fmt}: checked steps against 64 bits over the cache: {worst:.1e} of the largest value")
    return worst


def run(argv: list[str] | None = None) -> int:
    """The command: 0 where the checked steps hold to 64 bits, else 1."""
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--fmt", choices=("int8", "fp8"), default="int8")
    ap.add_argument("--chunk", type=int, default=256, help="tokens of a prompt that a step takes")
    a = ap.parse_args(argv)
    if a.chunk < 1:
        ap.error("--chunk must be 1 or more")
    return 0 if main(a.fmt, a.chunk) <= 2.0 ** -7 else 1  # (a NaN is no success)


if __name__ == "__main__":
    sys.exit(run())
