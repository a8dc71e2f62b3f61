"""The prompt's way through an attention layer over the 8-bit cache, as a
serving program runs it through the public entry points.

A case is a dict of plain values; its "kind" names the operator:

  plan    a step's tables from the requests' lengths: pages of sequences that
          are over go back to the list of free ones, new tokens' pages are
          taken from it; offsets, positions and cache slots of the new rows
  rope    queries and keys turned by their positions, their heads normed in
          the same pass where the layer has such weights
  prompt  whole prompts attend themselves, causal, packed one after the other
  chunk   new tokens of each sequence attend what the cache holds of it, and
          themselves, causal

The cache: pages of 64 tokens; keys [page][head][64][Dp], values
[page][head][Dp][64] with the tokens of a row in `_SLOT` order, one byte a
value, Dp = D rounded up to 32 (zeros past D); fp32 scales [page][head][64].
"""
import math
import random

import torch

own = False

PAGE = 64
# Place of token t of a page within a row of values.
_SLOT = [16 * ((t >> 2) & 3) + 8 * (t >> 5) + 4 * ((t >> 4) & 1) + (t & 3) for t in range(PAGE)]


def listed():
    return [
        # a decode step of many requests, one token each, some of them over: the tables' smallest call
        dict(name="plan_decode", kind="plan", B=256, n=1, start=3000, width=128, over=0.04, spare=40),
        # chunks of a prefill are admitted beside running requests, on a list that runs short of pages
        dict(name="plan_prompts", kind="plan", B=48, n=2048, start=5000, width=512, over=0.1, spare=900),
        # a decode step's rows, positions far out: the smallest turn
        dict(name="rope_token", kind="rope", dtype="bf16", n=16, reach=131072, Hq=32, Hkv=8, D=128, rot=128,
             pairs="half", norm=False, theta=500000.0, scaling="none", factor=1.0),
        # one prompt's chunk, heads normed before they are turned
        dict(name="rope_chunk", kind="rope", dtype="bf16", n=2048, reach=8192, Hq=32, Hkv=8, D=128, rot=128,
             pairs="half", norm=True, theta=1000000.0, scaling="none", factor=1.0),
        # part of an odd head, adjacent pairs, fp32, positions interpolated
        dict(name="rope_part", kind="rope", dtype="f32", n=777, reach=16384, Hq=15, Hkv=5, D=80, rot=40,
             pairs="adjacent", norm=True, theta=10000.0, scaling="linear", factor=4.0),
        # eight whole prompts: the most bytes, frequencies stretched by parts
        dict(name="rope_prompts", kind="rope", dtype="bf16", n=32768, reach=65536, Hq=32, Hkv=8, D=128, rot=128,
             pairs="half", norm=False, theta=10000.0, scaling="yarn", factor=16.0),
        # a few short questions: latency
        dict(name="prompt_short", kind="prompt", B=4, n=200, ragged=True, Hq=32, Hkv=8, D=128),
        # a batch of prompts packed, of different lengths
        dict(name="prompt_batch", kind="prompt", B=16, n=2048, ragged=True, Hq=32, Hkv=8, D=128),
        # one long document: the most arithmetic
        dict(name="prompt_long", kind="prompt", B=1, n=16384, ragged=False, Hq=32, Hkv=8, D=128),
        # odd head size and group, ragged prefixes of which some are empty
        dict(name="chunk_odd", kind="chunk", fmt="int8", B=6, n=190, L=1100, ragged=True, Hq=15, Hkv=5, D=80),
        # a mixed step: most sequences decode a token, some prefill a chunk
        dict(name="chunk_mixed", kind="chunk", fmt="int8", B=24, n=512, L=4096, ragged=True, Hq=32, Hkv=8, D=128),
        # a follow-up question over a long cached document
        dict(name="chunk_long", kind="chunk", fmt="fp8", B=1, n=512, L=32768, ragged=False, Hq=64, Hkv=8, D=128),
    ]


# ---- drawn cases ------------------------------------------------------------

def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    """One more case of the ranges the listed ones stand for, at no more than
    the cost of the largest of them."""
    kind = rng.choice(["plan", "rope", "rope", "prompt", "prompt", "chunk", "chunk", "chunk"])
    if kind == "plan":
        B = _log_int(rng, 1, 512)
        n = rng.choice([1, _log_int(rng, 1, 98304 // B)])
        return dict(kind=kind, B=B, n=n, start=_log_int(rng, 1, 16000), width=rng.choice([256, 300, 512, 1024]),
                    over=rng.choice([0.0, 0.1, 0.3]), spare=_log_int(rng, 1, 2000))
    Hkv, D = rng.choice([1, 2, 3, 4, 5, 8, 8, 8, 16]), rng.choice([40, 64, 64, 80, 96, 128, 128, 128, 128, 192, 256])
    Hq = Hkv * rng.choice([1, 1, 2, 3, 4, 4, 5, 7, 8, 8])
    if kind == "rope":
        dtype = rng.choice(["bf16", "bf16", "f32"])
        return dict(kind=kind, dtype=dtype, n=_log_int(rng, 1, min(32768, 32768 * 40 * 128 // ((Hq + Hkv) * D))),
                    reach=_log_int(rng, 500, 1000000), Hq=Hq, Hkv=Hkv, D=D, rot=rng.choice([D, D, D // 2, D - 2]),
                    pairs=rng.choice(["half", "half", "adjacent"]), norm=rng.random() < 0.5,
                    theta=rng.choice([10000.0, 500000.0, 1000000.0]),
                    scaling=rng.choice(["none", "linear", "ntk", "yarn"]), factor=rng.choice([2.0, 4.0, 16.0]))
    B, ragged = _log_int(rng, 1, 32), rng.random() < 0.7
    # scores of the plain form, at most those of prompt_long
    top = 32 * 16384 * 16384 * 128 // (B * Hq * max(D, 128))
    if kind == "prompt":
        return dict(kind=kind, B=B, n=_log_int(rng, 1, min(16384, int(top ** 0.5))), ragged=ragged, Hq=Hq, Hkv=Hkv,
                    D=D)
    n = _log_int(rng, 1, min(4096, int((top / 4) ** 0.5)))
    return dict(kind=kind, fmt=rng.choice(["int8", "fp8"]), B=B, n=n, L=_log_int(rng, 16, min(65536, top // (4 * n))),
                ragged=ragged, Hq=Hq, Hkv=Hkv, D=D)


# ---- a case's lengths -------------------------------------------------------

def _spread(B, top, ragged, least=0):
    """B lengths up to `top`: all `top`, or spread between `least` and it (the
    first the longest, every fifth the least)."""
    if not ragged:
        return [top] * B
    return [top if s == 0 else least if s % 5 == 4 else least + int((top - least) * ((s * 0.6180339887) % 1.0))
            for s in range(B)]


def _lengths(case):
    """(tokens each sequence holds before the call, new tokens of each; in a
    plan -1 where the sequence is over)."""
    B, n = case["B"], case["n"]
    if case["kind"] == "plan":
        every = int(1 / case["over"]) if case["over"] else B + 1
        return (_spread(B, case["start"], True, 1),
                [-1 if s % every == every - 1 else t for s, t in enumerate(_spread(B, n, n > 1, 1))])
    new = _spread(B, n, case["ragged"], 1)
    if case["kind"] == "prompt":
        return [0] * B, new
    if case["ragged"]:  # a step of a serving engine: two of three sequences only decode
        new = [t if s % 3 == 0 else 1 for s, t in enumerate(new)]
    # (the longest prefix is not the longest chunk's)
    return _spread(B, case["L"], case["ragged"])[::-1], new


# ---- inputs -----------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _heads(g, shape):
    """Keys and values: unit normal, each channel of each head with a gain of
    its own, a few channels much larger."""
    H, D = shape[-2:]
    gain = torch.exp(0.5 * torch.randn((H, D), generator=g, device="cuda"))
    gain = torch.where(torch.rand((H, D), generator=g, device="cuda") < 0.02, gain * 6, gain)
    return torch.randn(shape, generator=g, device="cuda").mul_(gain)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _sums(n):
    """Offsets of the sequences' rows: n[0], n[0] + n[1], ... after a zero."""
    out = [0]
    for x in n:
        out.append(out[-1] + x)
    return out


class _Cache:
    """A paged cache that holds random tokens, and the sequences' page lists."""

    def __init__(self, g, case, tokens, seed):
        B, H, D = case["B"], case["Hkv"], case["D"]
        Dp = (D + 31) // 32 * 32
        self.width = max(1, max(-(-t // PAGE) for t in tokens))
        self.pages = sum(-(-t // PAGE) for t in tokens) + 3
        order = random.Random(seed).sample(range(self.pages), self.pages)
        table, at = [], 0
        for t in tokens:
            n = -(-t // PAGE)
            table.append(order[at:at + n] + [-1] * (self.width - n))
            at += n
        self.table = _ints(table).view(B, self.width)
        self.slot = torch.tensor(_SLOT, device="cuda")
        self.k = torch.zeros((self.pages, H, PAGE, Dp), dtype=torch.uint8, device="cuda")
        self.v = torch.zeros((self.pages, H, Dp, PAGE), dtype=torch.uint8, device="cuda")
        codes, self.ks = self._quantize(_heads(g, (self.pages, PAGE, H, D)), case["fmt"])
        self.k[..., :D] = codes.transpose(1, 2)
        self.ks = self.ks.transpose(1, 2).contiguous()
        codes, self.vs = self._quantize(_heads(g, (self.pages, PAGE, H, D)), case["fmt"])
        self.v[:, :, :D, self.slot] = codes.permute(0, 2, 3, 1)
        self.vs = self.vs.transpose(1, 2).contiguous()

    @staticmethod
    def _quantize(x, fmt):
        scale = x.abs().amax(-1) / (127.0 if fmt == "int8" else 448.0)
        y = x / scale[..., None]
        if fmt == "int8":
            return y.round().to(torch.int8).view(torch.uint8), scale
        return y.to(torch.float8_e4m3fn).view(torch.uint8), scale


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case=case)
    if case["kind"] == "plan":
        return _prepare_plan(s, case, seed)
    if case["kind"] == "rope":
        return _prepare_rope(s, case, g, seed)
    held, new = _lengths(case)
    H, D, B, Hq = case["Hkv"], case["D"], case["B"], case["Hq"]
    offs, n = _ints(_sums(new)), sum(new)
    s.update(offsets=offs, start=_ints(held), n=n, new=max(new), cache=None, scale=D ** -0.5)
    # the sequence and the place in it of every new row, for the plain form
    s["seq"] = torch.repeat_interleave(torch.arange(B, device="cuda"), _ints(new).long())
    s["nth"] = torch.arange(n, device="cuda") - offs[s["seq"]]
    if case["kind"] == "chunk":
        s["cache"] = _Cache(g, case, held, seed)
    # one row of the fused projection's output holds queries, keys and values
    wide = torch.empty((n, (Hq + 2 * H) * D), dtype=torch.bfloat16, device="cuda")
    s["q"], s["k"], s["v"] = wide.split([Hq * D, H * D, H * D], dim=1)
    s["q"].copy_(torch.randn((n, Hq * D), generator=g, device="cuda").mul_(2))
    s["k"].copy_(_heads(g, (n, H, D)).view(n, -1))
    s["v"].copy_(_heads(g, (n, H, D)).view(n, -1))
    if own:
        from longhornai_amd import ops
        c = s["cache"]
        s["handle"] = c and ops.KvCache(case["fmt"], c.pages, H, D, c.k, c.v, c.ks, c.vs)
        s["ws"] = ops.prefill_workspace(B, n, Hq, H, D)
    return s


def _prepare_plan(s, case, seed):
    held, new = _lengths(case)
    r = random.Random(seed)
    # another seed: the same requests in another order, on other pages
    order = r.sample(range(case["B"]), case["B"])
    held, new = [held[i] for i in order], [new[i] for i in order]
    need = [min(case["width"], -(-t // PAGE)) for t in held]
    pages = sum(need) + case["spare"]
    ids, at, table = r.sample(range(pages), pages), 0, []
    for k in need:
        table.append(ids[at:at + k] + [-1] * (case["width"] - k))
        at += k
    s.update(held=_ints(held), new=_ints(new), table=_ints(table), pages=pages, n=sum(t for t in new if t > 0) + 3,
             # the list of free pages is a stack: the first `left` entries of it
             free=_ints(ids[at:] + [0] * at), left=_ints([case["spare"], 0]))
    return s


def _frequencies(case):
    """Radians a position of each pair, in 64 bits."""
    rot, f = case["rot"], case["factor"]
    theta = case["theta"] * (f ** (rot / (rot - 2)) if case["scaling"] == "ntk" else 1.0)
    freq = theta ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    if case["scaling"] == "linear":
        freq = freq / f
    if case["scaling"] == "yarn":  # pairs of under one turn in the first 4096 positions are stretched, of over 32 not
        keep = ((4096 * freq / (2 * math.pi) - 1) / (32 - 1)).clamp(0, 1)
        freq = freq / f * (1 - keep) + freq * keep
    return freq


def _gain(case):
    return 0.1 * math.log(case["factor"]) + 1 if case["scaling"] == "yarn" else 1.0


def _prepare_rope(s, case, g, seed):
    n, Hq, H, D = case["n"], case["Hq"], case["Hkv"], case["D"]
    dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    wide = torch.empty((n, (Hq + 2 * H) * D), dtype=dtype, device="cuda")
    s["q"], s["k"], _ = wide.split([Hq * D, H * D, H * D], dim=1)
    s["q"].copy_(torch.randn((n, Hq * D), generator=g, device="cuda").mul_(2))
    s["k"].copy_(_heads(g, (n, H, D)).view(n, -1))
    # runs of positions, as sequences have them
    r, at = random.Random(seed), 0
    s["pos"] = torch.empty(n, dtype=torch.int32, device="cuda")
    while at < n:
        run, first = min(n - at, _log_int(r, 1, max(2, n))), r.randrange(case["reach"])
        s["pos"][at:at + run] = torch.arange(first, first + run, device="cuda")
        at += run
    s["qw"] = s["kw"] = None
    if case["norm"]:
        s["qw"], s["kw"] = ((1 + 0.3 * torch.randn(D, generator=g, device="cuda")).to(dtype) for _ in range(2))
    if own:
        from longhornai_amd import ops
        s["plan"] = ops.rope_plan(D, rot_dim=case["rot"], theta=case["theta"], interleaved=case["pairs"] == "adjacent",
                                  scaling=None if case["scaling"] == "none" else case["scaling"],
                                  factor=case["factor"], original=4096)
    else:
        s["freq"] = _frequencies(case)
    return s


# ---- one pass ---------------------------------------------------------------

def run(s):
    kind = s["case"]["kind"]
    if kind == "plan":
        return _own_plan(s) if own else _plain_plan(s)
    if kind == "rope":
        return _own_rope(s) if own else _plain_rope(s)
    return _own_attend(s) if own else _plain_attend(s)


def _bits(x):
    """bf16 as the 16-bit patterns that the library's entry points take."""
    return x.view(torch.int16) if x is not None and x.dtype == torch.bfloat16 else x


def _own_plan(s):
    from longhornai_amd import ops
    p = ops.kv_plan(s["held"], s["new"], s["free"], s["left"], s["table"], s["n"])
    return dict(offsets=p.offsets, positions=p.positions, slots=p.slots, left=p.left, table=s["table"], free=s["free"])


def _own_rope(s):
    from longhornai_amd import ops
    q, k = ops.rope(s["plan"], _bits(s["q"]), _bits(s["k"]), s["pos"], q_weight=_bits(s["qw"]),
                    k_weight=_bits(s["kw"]), eps=1e-6)
    return (q.view(torch.bfloat16), k.view(torch.bfloat16)) if q.dtype == torch.int16 else (q, k)


def _own_attend(s):
    from longhornai_amd import ops
    q, k, v, case = _bits(s["q"]), _bits(s["k"]), _bits(s["v"]), s["case"]
    if case["kind"] == "prompt":
        out = ops.attn_prompt(q, k, v, s["offsets"], case["D"], scale=s["scale"], workspace=s["ws"])
    else:
        out = ops.kv_prefill(s["handle"], q, s["offsets"], s["start"], s["cache"].table, k, v, scale=s["scale"],
                             workspace=s["ws"])
    return out.view(torch.bfloat16)


def _plain_plan(s):
    table, free, B, W, P = s["table"], s["free"], s["case"]["B"], s["case"]["width"], s["pages"]
    held, new = s["held"].long().clamp(0, W * PAGE), s["new"].long()
    # rows
    offsets = torch.cat([new.new_zeros(1), new.clamp(min=0).cumsum(0)]).clamp(max=s["n"])
    new, over = offsets[1:] - offsets[:-1], new < 0
    # pages of sequences that are over go on the stack, by sequence and page
    p = torch.arange(W, device="cuda")
    had, wants = (held + PAGE - 1) // PAGE, ((held + new + PAGE - 1) // PAGE).clamp(max=W)
    back = over[:, None] & (p < had[:, None]) & (table >= 0) & (table < P)
    at = s["left"][0] + back.flatten().cumsum(0) - 1
    back = back.flatten() & (at < P)
    free.copy_(torch.cat([free, free.new_zeros(1)]).scatter_(0, torch.where(back, at, P), table.flatten())[:P])
    have = s["left"][0] + back.sum()
    # new pages come off it, in the same order
    take = (~over[:, None] & (p >= had[:, None]) & (p < wants[:, None])).flatten()
    nth = take.cumsum(0) - 1
    got = torch.where(nth < have, free[(have - 1 - nth).clamp(min=0)], torch.full_like(free[:1], -1))
    table.copy_(torch.where(take, got, table.flatten()).view(B, W))
    asked = take.sum()
    left = torch.stack([(have - asked).clamp(min=0), (asked - have).clamp(min=0)]).int()
    # rows: the last sequence whose first row is not behind the row
    row = torch.arange(s["n"], device="cuda")
    seq = (torch.searchsorted(offsets, row, right=True) - 1).clamp(max=B - 1)
    at = held[seq] + row - offsets[seq]
    there = row < offsets[B]
    page = table[seq, (at // PAGE).clamp(max=W - 1)]
    some = there & (at < W * PAGE) & (page >= 0) & (page < P)
    slots = torch.where(some, page.long() * PAGE + at % PAGE, torch.full_like(at, -1))
    return dict(offsets=offsets.int(), positions=torch.where(there, at, torch.full_like(at, -1)).int(), slots=slots,
                left=left, table=table, free=free)


def _plain_rope(s):
    case = s["case"]
    rot, D = case["rot"], case["D"]
    angle = s["pos"].double()[:, None] * s["freq"]
    cos, sin = (f(angle).mul(_gain(case)).float()[:, None, :] for f in (torch.cos, torch.sin))

    def turned(x, weight):
        y = x.float().view(len(x), -1, D)
        if weight is not None:
            y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * weight.float()
        if case["pairs"] == "half":
            a, b = y[..., :rot // 2], y[..., rot // 2:rot]
            parts = [a * cos - b * sin, b * cos + a * sin]
        else:
            a, b = y[..., 0:rot:2], y[..., 1:rot:2]
            parts = [torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(2)]
        return torch.cat(parts + [y[..., rot:]], dim=-1).to(x.dtype)

    return turned(s["q"], s["qw"]), turned(s["k"], s["kw"])


def _values(codes, fmt):
    return codes.view(torch.int8 if fmt == "int8" else torch.float8_e4m3fn).float()


def _plain_attend(s):
    case, c = s["case"], s["cache"]
    B, T, H, D, Hq = case["B"], s["new"], case["Hkv"], case["D"], case["Hq"]
    G, seq, nth = Hq // H, s["seq"], s["nth"]

    def padded(x, heads):
        """The sequences' new rows beside one another: [B, heads, T, D]."""
        y = torch.zeros((B, T, heads, D), dtype=torch.float32, device="cuda")
        y[seq, nth] = x.float().view(-1, heads, D)
        return y.transpose(1, 2)

    q, k, v = padded(s["q"], Hq).reshape(B, H, G * T, D), padded(s["k"], H), padded(s["v"], H)
    i = torch.arange(T, device="cuda")
    seen = (i <= i[:, None]).expand(B, T, T)
    if c is not None:
        fmt, W, table = case["fmt"], c.width * PAGE, c.table.clamp(min=0).long()
        kc = (_values(c.k[table], fmt) * c.ks[table][..., None]).transpose(1, 2).reshape(B, H, W, -1)[..., :D]
        vc = (_values(c.v[table][..., c.slot], fmt) * c.vs[table][..., None, :]).permute(0, 2, 1, 4, 3)
        k, v = torch.cat([kc, k], dim=2), torch.cat([vc.reshape(B, H, W, -1)[..., :D], v], dim=2)
        held = torch.arange(W, device="cuda") < s["start"][:, None]
        seen = torch.cat([held[:, None, :].expand(B, T, W), seen], dim=2)
    x = torch.matmul(q, k.transpose(2, 3)).mul_(s["scale"])
    x.view(B, H, G, T, -1).masked_fill_(~seen[:, None, None], -math.inf)
    p = x.sub_(x.amax(-1, keepdim=True)).exp_()  # (every row sees itself)
    o = torch.matmul(p, v).div_(p.sum(-1, keepdim=True))
    return o.view(B, H * G, T, D).transpose(1, 2)[seq, nth].to(torch.bfloat16)


# ---- work and exact values --------------------------------------------------

def work(case):
    held, new = (0, 0) if case["kind"] == "rope" else _lengths(case)
    if case["kind"] == "plan":
        rows, pages = sum(t for t in new if t > 0), sum(-(-t // PAGE) for t in held)
        # lengths and counts in, offsets out; a position and a slot a row; pages that come or go, in list and table
        moved = sum(-(-t // PAGE) if n < 0 else -(-(t + n) // PAGE) - -(-t // PAGE) for t, n in zip(held, new))
        return {"bytes": 12 * case["B"] + 12 * rows + 8 * min(moved, pages + case["spare"]), "flops": rows + moved}
    H, D, Hq = case["Hkv"], case["D"], case["Hq"]
    if case["kind"] == "rope":
        values = case["n"] * (Hq + H) * D
        return {"bytes": 2 * values * (2 if case["dtype"] == "bf16" else 4) + 4 * case["n"],
                "flops": 3 * values + (4 * values if case["norm"] else 0)}
    cached = 2 * H * (D + 4) if case["kind"] == "chunk" else 0  # codes and scales of one token
    return {"bytes": sum(held) * cached + sum(new) * 2 * D * (2 * Hq + 2 * H),
            "flops": sum(4 * Hq * D * (t * h + t * (t + 1) // 2) for h, t in zip(held, new))}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "plan":
        return _exact_plan(s)
    if case["kind"] == "rope":
        return _exact_rope(s)
    return _exact_attend(s)


def _exact_plan(s):
    held, new, table, free = (s[k].tolist() for k in ("held", "new", "table", "free"))
    stack, P, W = free[:s["left"][0].item()], s["pages"], s["case"]["width"]
    for h, n, row in zip(held, new, table):
        if n < 0:
            stack += [p for p in row[:min(W, -(-h // PAGE))] if 0 <= p < P]
    free[:len(stack)] = stack
    offsets, missing = [0], 0
    positions, slots = [-1] * s["n"], [-1] * s["n"]
    for h, n, row in zip(held, new, table):
        first = offsets[-1]
        offsets.append(first + max(n, 0))
        for p in range(-(-h // PAGE), min(W, -(-(h + n) // PAGE)) if n > 0 else 0):
            missing += not stack
            row[p] = stack.pop() if stack else -1
        for i in range(max(n, 0)):
            at = positions[first + i] = h + i
            if at < W * PAGE and 0 <= row[at // PAGE] < P:
                slots[first + i] = row[at // PAGE] * PAGE + at % PAGE
    return dict(offsets=_ints(offsets), positions=_ints(positions), slots=torch.tensor(slots, device="cuda"),
                left=_ints([len(stack), missing]), table=_ints(table), free=_ints(free))


def _exact_rope(s):
    case = s["case"]
    rot, D, n = case["rot"], case["D"], case["n"]
    # each pair a complex number
    angle = s["pos"].double()[:, None] * _frequencies(case)
    turn = torch.polar(torch.full_like(angle, _gain(case)), angle)[:, None]
    out = []
    for x, w in ((s["q"], s["qw"]), (s["k"], s["kw"])):
        x = x.double().view(n, -1, D)
        if w is not None:
            x = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
        half = case["pairs"] == "half"
        z = torch.complex(x[..., :rot // 2], x[..., rot // 2:rot]) if half else \
            torch.view_as_complex(x[..., :rot].unflatten(-1, (-1, 2)).contiguous())
        z = torch.view_as_real(z * turn)
        x = x.clone()
        x[..., :rot] = (z.transpose(-1, -2) if half else z).flatten(-2)
        out.append(x)
    return tuple(out)


def _e4m3_table():
    """The 256 values of e4m3, by its definition."""
    def value(c):
        e, m = c >> 3 & 15, c & 7
        if e == 15 and m == 7:
            return math.nan
        x = m * 2.0 ** -9 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        return -x if c >> 7 else x
    return torch.tensor([value(c) for c in range(256)], dtype=torch.float64, device="cuda")


def _cached64(s, which, b, L):
    """The first L tokens of sequence b as the cache holds them: [L, H, D]."""
    case, c = s["case"], s["cache"]
    codes, scales = (c.k, c.ks) if which == "k" else (c.v, c.vs)
    pages = c.table[b, :(L + PAGE - 1) // PAGE].long()
    x = codes[pages]
    x = x.permute(0, 2, 1, 3) if which == "k" else x.permute(0, 3, 1, 2).index_select(1, c.slot)
    x = x[..., :case["D"]].flatten(0, 1)
    table = _e4m3_table() if case["fmt"] == "fp8" else \
        torch.tensor([u - 256 if u > 127 else u for u in range(256)], dtype=torch.float64, device="cuda")
    return (table[x.int()] * scales[pages].permute(0, 2, 1).flatten(0, 1).double()[..., None])[:L]


def _exact_attend(s):
    case = s["case"]
    held, new = _lengths(case)
    H, D, offs, Hq = case["Hkv"], case["D"], _sums(new), case["Hq"]
    G = Hq // H
    out = torch.zeros((s["n"], Hq, D), dtype=torch.float64, device="cuda")
    for b in range(case["B"]):
        L, T, at = held[b], new[b], slice(offs[b], offs[b + 1])
        hidden = torch.ones((T, L + T), dtype=torch.bool, device="cuda").triu(L + 1)
        k64, v64 = (_cached64(s, w, b, L) if L else torch.zeros((0, H, D), dtype=torch.float64, device="cuda")
                    for w in "kv")
        for h in range(H):
            k = torch.cat([k64[:, h], s["k"][at].double().view(T, H, D)[:, h]])
            v = torch.cat([v64[:, h], s["v"][at].double().view(T, H, D)[:, h]])
            q = s["q"][at].double().view(T, H, G, D)[:, h].transpose(0, 1).reshape(G * T, D)
            x = (q @ k.T.contiguous() * s["scale"]).view(G, T, L + T).masked_fill_(hidden, -math.inf)
            o = torch.softmax(x, -1).view(G * T, L + T) @ v
            out[at, h * G:(h + 1) * G] = o.view(G, T, D).transpose(0, 1)
            del x, o
    return out
