"""The 8-bit key/value cache and the attention that reads it, as a serving
program runs them through the public entry points.

A case is a dict of plain values; its "kind" names the operator:

  store   new tokens' keys and values quantized into the paged cache, and the
          written tokens read back (what a prefill chunk does before it
          attends what the cache holds)
  read    a range of every sequence's cached tokens read back
  attend  drafted tokens (a tree each, one token in plain decode) attend the
          cached tokens and their own ancestors

The cache: pages of 64 tokens; keys [page][head][64][Dp], values
[page][head][Dp][64] with the tokens of a row in `_SLOT` order, one byte a
value, Dp = D rounded up to 32 (zeros past D); fp32 scales [page][head][64].
Codes and scales follow the library's per-row rule: scale = max|x| / 127 (448
for e4m3; 1 for a row of zeros), code = x * (1 / scale) saturated and rounded
to nearest even (e4m3: zero below 2^-9).
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
        # a decode step's new tokens, 16 sequences: the smallest write
        dict(name="store_token", kind="store", fmt="int8", dtype="bf16", B=16, n=1, start=700, ragged=True, pick=0,
             Hkv=8, D=128),
        # the accepted tokens of 24 drafted trees, picked out of all drafted rows; fp32 rows, odd head size
        dict(name="store_accepted", kind="store", fmt="fp8", dtype="f32", B=24, n=5, start=333, ragged=True, pick=16,
             Hkv=5, D=80),
        # one chunk of a chunked prefill, starting inside a page
        dict(name="store_chunk", kind="store", fmt="int8", dtype="bf16", B=1, n=2048, start=1001, ragged=False,
             pick=0, Hkv=8, D=128),
        # eight whole prompts: the largest write
        dict(name="store_prompts", kind="store", fmt="fp8", dtype="bf16", B=8, n=4096, start=0, ragged=False, pick=0,
             Hkv=8, D=128),
        # a shared prefix pulled out of the cache for a prefill's own attention
        dict(name="read_prefix", kind="read", fmt="int8", dtype="bf16", B=1, n=16384, start=0, ragged=False, Hkv=8,
             D=128),
        # tails of many sequences, ragged, to fp32
        dict(name="read_ragged", kind="read", fmt="fp8", dtype="f32", B=24, n=1900, start=37, ragged=True, Hkv=4,
             D=96),
        # single-stream decode over a short context: the smallest attention, latency
        dict(name="decode_one", kind="attend", fmt="int8", B=1, T=1, L=500, ragged=False, Hq=32, Hkv=8, D=128),
        # batched decode, ragged lengths
        dict(name="decode_batch", kind="attend", fmt="fp8", B=64, T=1, L=4096, ragged=True, Hq=32, Hkv=8, D=128),
        # long contexts, few sequences: the most bytes
        dict(name="decode_long", kind="attend", fmt="int8", B=4, T=1, L=131072, ragged=False, Hq=32, Hkv=8, D=128),
        # verification of small drafted trees in a batch
        dict(name="tree_batch", kind="attend", fmt="int8", B=8, T=12, L=2500, ragged=True, Hq=64, Hkv=8, D=128),
        # widest trees: the most arithmetic
        dict(name="tree_wide", kind="attend", fmt="fp8", B=4, T=64, L=8192, ragged=False, Hq=64, Hkv=8, D=128),
        # odd head size and group, sequences of which some have nothing cached yet
        dict(name="tree_odd", kind="attend", fmt="int8", B=6, T=7, L=1100, ragged=True, Hq=15, Hkv=5, D=80),
    ]


# ---- drawn cases ------------------------------------------------------------

def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the ranges the listed ones stand for, at no more than
    the cost of the largest of them."""
    kind = rng.choice(["store", "store", "read", "attend", "attend", "attend", "attend"])
    case = dict(kind=kind, fmt=rng.choice(["int8", "fp8"]))
    Hkv, D = rng.choice([1, 2, 3, 4, 5, 8, 8, 8, 16]), rng.choice([40, 64, 64, 80, 96, 128, 128, 128, 128, 192, 256])
    if kind != "attend":
        case.update(dtype=rng.choice(["bf16", "bf16", "f32"]), B=_log_int(rng, 1, 64), ragged=rng.random() < 0.6,
                    start=rng.choice([0, _log_int(rng, 1, 4000)]), Hkv=Hkv, D=D)
        case["n"] = _log_int(rng, 1, max(1, min(16384, 8 * 4096 * 8 * 128 // (case["B"] * Hkv * D))))
        if kind == "store":
            case["pick"] = case["n"] + _log_int(rng, 1, 16) if case["n"] <= 16 and rng.random() < 0.5 else 0
        return case
    group = rng.choice([1, 1, 2, 3, 4, 4, 5, 7, 8, 8, 16])
    T = rng.choice([1, 1, _log_int(rng, 1, 64), _log_int(rng, 2, 64)])
    B = _log_int(rng, 1, 64)
    # at most the bytes of decode_long and the arithmetic of tree_wide
    top = min(4 * 131072 * 8 * 128 // (B * Hkv * D), 4 * 64 * 64 * 8192 * 128 // (B * Hkv * group * T * D))
    L = _log_int(rng, 16, max(17, min(131072, top)))
    case.update(B=B, T=T, L=L, ragged=rng.random() < 0.6, Hq=Hkv * group, Hkv=Hkv, D=D)
    return case


# ---- a case's lengths -------------------------------------------------------

def _spread(B, top, ragged, least=0):
    """B lengths up to `top`: all `top`, or spread between `least` and it (the
    first the longest, every fifth the least)."""
    if not ragged:
        return [top] * B
    return [top if s == 0 else least if s % 5 == 4 else least + int((top - least) * ((s * 0.6180339887) % 1.0))
            for s in range(B)]


def _lengths(case):
    """(tokens each sequence holds before the call, new tokens of each)."""
    B = case["B"]
    if case["kind"] == "attend":
        T = case["T"]
        return _spread(B, case["L"], case["ragged"]), _spread(B, T, case["ragged"] and T > 2, 1)
    start = _spread(B, case["start"], case["ragged"])
    return start, _spread(B, case["n"], case["ragged"] and case["n"] > 1, 1)


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


def _pad(D):
    return (D + 31) // 32 * 32


def _quantize(x, fmt):
    """Codes (bytes) and scales of the last axis, by the library's rule."""
    amax = x.abs().amax(-1)
    # tensors over tensors: a division by a Python number multiplies by its rounded reciprocal
    one, top = torch.ones_like(amax), torch.full_like(amax, 127.0 if fmt == "int8" else 448.0)
    scale = torch.where(amax > 0, amax / top, one)
    y = x * (one / scale)[..., None]
    if fmt == "int8":
        return y.clamp(-127, 127).round().to(torch.int8).view(torch.uint8), scale
    y = torch.where(y.abs() < 2.0 ** -9, torch.zeros_like(y), y.clamp(-448, 448))
    return y.to(torch.float8_e4m3fn).view(torch.uint8), scale


def _values(codes, fmt):
    return codes.view(torch.int8 if fmt == "int8" else torch.float8_e4m3fn).float()


class _Cache:
    """A paged cache that holds random tokens, and the sequences' page lists."""

    def __init__(self, g, case, tokens, spare, seed):
        B, H, D, Dp = case["B"], case["Hkv"], case["D"], _pad(case["D"])
        self.width = max(1, max(-(-t // PAGE) for t in tokens))
        self.pages = sum(-(-t // PAGE) for t in tokens) + spare
        order = random.Random(seed).sample(range(self.pages), self.pages)
        table, at = [], 0
        for t in tokens:
            n = -(-t // PAGE)
            table.append(order[at:at + n] + [-1] * (self.width - n))
            at += n
        self.table = torch.tensor(table, dtype=torch.int32, device="cuda").view(B, self.width)
        self.k = torch.zeros((self.pages, H, PAGE, Dp), dtype=torch.uint8, device="cuda")
        self.v = torch.zeros((self.pages, H, Dp, PAGE), dtype=torch.uint8, device="cuda")
        self.slot = torch.tensor(_SLOT, device="cuda")
        codes, self.ks = _quantize(_heads(g, (self.pages, PAGE, H, D)), case["fmt"])
        self.k[..., :D] = codes.transpose(1, 2)
        self.ks = self.ks.transpose(1, 2).contiguous()
        codes, self.vs = _quantize(_heads(g, (self.pages, PAGE, H, D)), case["fmt"])
        self.v[:, :, :D, self.slot] = codes.permute(0, 2, 3, 1)
        self.vs = self.vs.transpose(1, 2).contiguous()

    def handle(self, case):
        """The library's handle on these buffers."""
        from longhornai_amd import ops
        return ops.KvCache(case["fmt"], self.pages, case["Hkv"], case["D"], self.k, self.v, self.ks, self.vs)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _sums(n):
    """Offsets of the sequences' rows: n[0], n[0] + n[1], ... after a zero."""
    return [sum(n[:i]) for i in range(len(n) + 1)]


def _trees(n, seed):
    """Ancestor masks: bit j of a drafted token's word is set where the token
    j of the same tree is the token itself or above it."""
    r, words = random.Random(seed), []
    for T in n:
        tree = []
        for i in range(T):
            parent = r.choice([i - 1, i - 1, r.randrange(-1, i)]) if i else -1
            tree.append((tree[parent] if parent >= 0 else 0) | 1 << i)
        words += [w - (1 << 64) if w >> 63 else w for w in tree]
    return torch.tensor(words, dtype=torch.int64, device="cuda")


def prepare(case, seed):
    g = _gen(seed)
    held, new = _lengths(case)
    H, D, B = case["Hkv"], case["D"], case["B"]
    offs, n = _ints(_sums(new)), sum(new)
    s = dict(case=case, offsets=offs, start=_ints(held), n=n, new=max(new))
    # the sequence and the position of every new row, for the plain form
    s["seq"] = torch.repeat_interleave(torch.arange(B, device="cuda"), _ints(new).long())
    s["nth"] = torch.arange(n, device="cuda") - offs[s["seq"]]
    if case["kind"] == "attend":
        s["cache"] = _Cache(g, case, held, 3, seed)
        G = case["Hq"] // H
        # one row of the fused projection's output holds queries, keys and values
        wide = torch.empty((n, (case["Hq"] + 2 * H) * D), dtype=torch.bfloat16, device="cuda")
        q, k, v = wide.split([case["Hq"] * D, H * D, H * D], dim=1)
        q.copy_(torch.randn((n, H * G * D), generator=g, device="cuda").mul_(2))
        k.copy_(_heads(g, (n, H, D)).view(n, -1))
        v.copy_(_heads(g, (n, H, D)).view(n, -1))
        s.update(q=q, k=k, v=v, tree=_trees(new, seed), scale=D ** -0.5)
    else:
        s["cache"] = _Cache(g, case, [a + b for a, b in zip(held, new)], 3, seed)
    dtype = torch.bfloat16 if case.get("dtype") == "bf16" else torch.float32
    if case["kind"] == "store":
        rows = case["pick"] * B if case["pick"] else n
        s["k"], s["v"] = (_heads(g, (rows, H, D)).to(dtype).view(rows, H * D) for _ in range(2))
        s["rows"] = None
        if case["pick"]:
            r = random.Random(seed)
            s["rows"] = _ints([b * case["pick"] + i for b in range(B)
                               for i in sorted(r.sample(range(case["pick"]), new[b]))])
    if own:
        from longhornai_amd import ops
        s["handle"] = s["cache"].handle(case)
        if case["kind"] == "attend":
            s["ws"] = ops.kv_attn_workspace(s["handle"], B, s["n"], s["new"], s["cache"].width, case["Hq"])
    return s


# ---- one pass ---------------------------------------------------------------

def run(s):
    kind = s["case"]["kind"]
    if own:
        return _own_attend(s) if kind == "attend" else _own_cache(s, kind == "store")
    return _plain_attend(s) if kind == "attend" else _plain_cache(s, kind == "store")


def _bits(x):
    """bf16 as the 16-bit patterns that the library's entry points take."""
    return x.view(torch.int16) if x.dtype == torch.bfloat16 else x


def _own_cache(s, store):
    from longhornai_amd import ops
    case, table = s["case"], s["cache"].table
    if store:
        ops.kv_write(s["handle"], _bits(s["k"]), _bits(s["v"]), s["offsets"], s["start"], table, rows=s["rows"])
    bf16 = case["dtype"] == "bf16"
    k, v = ops.kv_read(s["handle"], s["offsets"], s["start"], table, s["n"], bf16=bf16)
    return (k.view(torch.bfloat16), v.view(torch.bfloat16)) if bf16 else (k, v)


def _own_attend(s):
    from longhornai_amd import ops
    out = ops.kv_attn(s["handle"], _bits(s["q"]), s["offsets"], s["start"], s["cache"].table, _bits(s["k"]),
                      _bits(s["v"]), tree=s["tree"], scale=s["scale"], max_new=s["new"], workspace=s["ws"])
    return out.view(torch.bfloat16)


def _plain_cache(s, store):
    case, c = s["case"], s["cache"]
    H, D, fmt = case["Hkv"], case["D"], case["fmt"]
    at = s["start"][s["seq"]] + s["nth"]
    page, tok = c.table[s["seq"], at // PAGE].long(), at % PAGE
    slot = c.slot[tok]
    if store:
        k, v = (x if s["rows"] is None else x[s["rows"]] for x in (s["k"], s["v"]))
        codes, c.ks[page, :, tok] = _quantize(k.view(-1, H, D).float(), fmt)
        c.k[page, :, tok, :D] = codes
        codes, c.vs[page, :, tok] = _quantize(v.view(-1, H, D).float(), fmt)
        c.v[page, :, :D, slot] = codes
    dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    k = _values(c.k[page, :, tok, :D], fmt) * c.ks[page, :, tok][..., None]
    v = _values(c.v[page, :, :D, slot], fmt) * c.vs[page, :, tok][..., None]
    return k.to(dtype), v.to(dtype)


def _plain_attend(s):
    case, c = s["case"], s["cache"]
    B, T, H, D, fmt = case["B"], s["new"], case["Hkv"], case["D"], case["fmt"]
    G = case["Hq"] // H
    seq, nth, table = s["seq"], s["nth"], c.table.clamp(min=0).long()
    W = c.width * PAGE

    def padded(x, heads):
        """The sequences' new rows beside one another: [B, heads, T, D]."""
        y = torch.zeros((B, T, heads, D), dtype=torch.float32, device="cuda")
        y[seq, nth] = x.float().view(-1, heads, D)
        return y.transpose(1, 2)

    # cached and new keys and values, [B, H, W + T, D]
    k = (_values(c.k[table], fmt) * c.ks[table][..., None]).transpose(1, 2).reshape(B, H, W, -1)[..., :D]
    v = (_values(c.v[table][..., c.slot], fmt) * c.vs[table][..., None, :]).permute(0, 2, 1, 4, 3)
    v = v.reshape(B, H, W, -1)[..., :D]
    k = torch.cat([k, padded(s["k"], H)], dim=2)
    v = torch.cat([v, padded(s["v"], H)], dim=2)
    q = padded(s["q"], case["Hq"]).reshape(B, H, G * T, D)
    x = torch.matmul(q, k.transpose(2, 3)) * s["scale"]
    # which of them a row of queries sees: cached tokens below the length, and its tree's bits
    bits = torch.zeros((B, T), dtype=torch.int64, device="cuda")
    bits[seq, nth] = s["tree"]
    below = torch.arange(W, device="cuda") < s["start"][:, None]
    above = (bits[:, :, None] >> torch.arange(T, device="cuda")) & 1
    seen = torch.cat([below[:, None, :].expand(B, T, W), above.bool()], dim=2)
    x = x.view(B, H, G, T, W + T).masked_fill(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
    o = torch.matmul(p.view(B, H, G * T, W + T), v).view(B, H, G, T, D)
    total = p.sum(-1)[..., None]
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return o.permute(0, 3, 1, 2, 4)[seq, nth].reshape(-1, case["Hq"], D).to(torch.bfloat16)


# ---- work and exact values --------------------------------------------------

def work(case):
    held, new = _lengths(case)
    H, D, n = case["Hkv"], case["D"], sum(new)
    row = 2 * H * D * (2 if case.get("dtype", "bf16") == "bf16" else 4)
    cached = 2 * H * (D + 4)  # codes and scales of one token
    if case["kind"] == "attend":
        return {"bytes": sum(held) * cached + n * (row + 2 * 2 * case["Hq"] * D),
                "flops": sum(4 * t * case["Hq"] * D * (h + (t + 1) // 2) for h, t in zip(held, new))}
    passes = 2 if case["kind"] == "store" else 1
    return {"bytes": passes * n * (row + cached), "flops": passes * 2 * n * H * D}


def _e4m3_table():
    """The 256 values of e4m3, by its definition."""
    def value(c):
        e, m = c >> 3 & 15, c & 7
        if e == 15 and m == 7:
            return math.nan
        x = m * 2.0 ** -9 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        return -x if c >> 7 else x
    return torch.tensor([value(c) for c in range(256)], dtype=torch.float64, device="cuda")


def _cached64(s, which, b, lo, hi):
    """Tokens lo .. hi of sequence b as the cache holds them: [hi - lo, H, D]."""
    case, c = s["case"], s["cache"]
    codes, scales = (c.k, c.ks) if which == "k" else (c.v, c.vs)
    pages = c.table[b, lo // PAGE:(hi + PAGE - 1) // PAGE].long()
    x = codes[pages]
    x = x.permute(0, 2, 1, 3) if which == "k" else x.permute(0, 3, 1, 2).index_select(1, c.slot)
    x = x[..., :case["D"]].flatten(0, 1)
    table = _e4m3_table() if case["fmt"] == "fp8" else \
        torch.tensor([u - 256 if u > 127 else u for u in range(256)], dtype=torch.float64, device="cuda")
    x = table[x.int()] * scales[pages].permute(0, 2, 1).flatten(0, 1).double()[..., None]
    first = lo // PAGE * PAGE
    return x[lo - first:hi - first]


def _stored64(x, fmt):
    """What a row of the cache stands for after it was given x.  The scale, its
    reciprocal and their product with x are 32-bit numbers by the rule: each
    is made in 64 bits and rounded to 32, so codes at a border are the rule's."""
    def r32(t):
        return t.float().double()
    amax = x.abs().amax(-1, keepdim=True)
    step = torch.where(amax > 0, r32(amax / (127.0 if fmt == "int8" else 448.0)), torch.ones_like(amax))
    y = r32(x * r32(1 / step))
    if fmt == "fp8":
        grid = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
        return torch.where(y.abs() < 2.0 ** -9, torch.zeros_like(y), torch.round(y / grid) * grid) * step
    return torch.round(y) * step


def exact(case, seed):
    s = prepare(case, seed)
    held, new = _lengths(case)
    H, D, offs = case["Hkv"], case["D"], _sums(new)
    if case["kind"] == "read":
        return tuple(torch.cat([_cached64(s, w, b, held[b], held[b] + new[b]) for b in range(case["B"])])
                     for w in "kv")
    if case["kind"] == "store":
        rows = slice(None) if s["rows"] is None else s["rows"].long()
        return tuple(_stored64(s[w][rows].double().view(-1, H, D), case["fmt"]) for w in "kv")
    G = case["Hq"] // H
    out = torch.zeros((s["n"], case["Hq"], D), dtype=torch.float64, device="cuda")
    for b in range(case["B"]):
        L, T, at = held[b], new[b], slice(offs[b], offs[b + 1])
        bits = s["tree"][at]
        seen = torch.ones((T, L + T), dtype=torch.bool, device="cuda")
        seen[:, L:] = (bits[:, None] >> torch.arange(T, device="cuda") & 1) == 1
        k64, v64 = (_cached64(s, w, b, 0, L) if L else torch.zeros((0, H, D), dtype=torch.float64, device="cuda")
                    for w in "kv")
        for h in range(H):
            k = torch.cat([k64[:, h], s["k"][at].double().view(T, H, D)[:, h]])
            v = torch.cat([v64[:, h], s["v"][at].double().view(T, H, D)[:, h]])
            q = s["q"][at].double().view(T, H, G, D)[:, h].reshape(T * G, D)
            x = (q @ k.T.contiguous() * s["scale"]).masked_fill(~seen.repeat_interleave(G, 0), -math.inf)
            out[at, h * G:(h + 1) * G] = (torch.softmax(x, -1) @ v).view(T, G, D)
    return out
