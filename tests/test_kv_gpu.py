"""The 8-bit key/value cache and attention over it on the GPU, against plain
64-bit numpy (tests/_kv.py) and, for the codes, the reference's per-row
quantizers: written codes, scales and values read back are bit-exact."""
import numpy as np
import pytest

from tests import _data as D
from tests import _kv

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(lib):
    from longhornai_amd import ops as _ops
    return _ops


def rng(seed):
    return np.random.default_rng(seed)


def offsets_of(n):
    return np.concatenate([[0], np.cumsum(n)]).astype(np.int32)


def quantize(oracle, fmt, x):
    return (oracle.fp8_quantize_per_row if fmt == "fp8" else oracle.q8_quantize_per_row)(x)


def wide(x):
    """fp32 values of rows given as fp32 or as bf16 bits."""
    return x if x.dtype == np.float32 else D.bf16_bits_to_f32(x)


def expect_write(oracle, c, k, v, offs, start, table, rows=None):
    """The write by its definition, into the host cache."""
    k, v = wide(k).reshape(len(k), c.H, c.D), wide(v).reshape(len(v), c.H, c.D)
    for s in range(len(start)):
        for i in range(offs[s], offs[s + 1]):
            r = i if rows is None else int(rows[i])
            at = c.find(table, s, int(start[s]) + i - int(offs[s]))
            if at is None or not 0 <= r < len(k):
                continue
            for h in range(c.H):
                qk, sk = quantize(oracle, c.fmt, k[r, h][None])
                qv, sv = quantize(oracle, c.fmt, v[r, h][None])
                c.put(*at[:1], h, at[1], qk.view(np.uint8)[0], qv.view(np.uint8)[0], sk[0], sv[0])


def same(ops, dev, c):
    assert np.array_equal(ops.host(dev.k), c.k), "key codes"
    assert np.array_equal(ops.host(dev.v), c.v), "value codes"
    assert np.array_equal(ops.host(dev.k_scales), c.ks), "key scales"
    assert np.array_equal(ops.host(dev.v_scales), c.vs), "value scales"


def make_rows(oracle, n, width, dtype, seed):
    x = rng(seed).standard_normal((n, width)).astype(np.float32)
    x *= np.exp(rng(seed + 1).standard_normal((n, 1))).astype(np.float32)
    return x if dtype == "f32" else D.to_bf16_bits(oracle, x)


# (new tokens, positions before them) of each sequence: empty ones, starts inside a page, pages crossed
LAYOUTS = {
    "token": ([1, 1, 1, 1, 1], [0, 63, 64, 200, 5]),
    "ragged": ([0, 130, 3, 0, 64, 1], [7, 61, 126, 0, 64, 191]),
    "chunk": ([300], [37]),
}


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("fmt,H,Dh", [("int8", 2, 128), ("fp8", 2, 128), ("int8", 3, 75), ("fp8", 1, 256), ("fp8", 5, 80),
                                      ("int8", 1, 40), ("int8", 2, 1), ("fp8", 2, 192), ("int8", 2, 64)])
def test_write_then_read(oracle, ops, fmt, H, Dh, dtype, layout):
    new, start = LAYOUTS[layout]
    offs, total = offsets_of(new), [a + b for a, b in zip(new, start)]
    pages = sum(-(-t // 64) for t in total) + 2
    c = _kv.HostCache(fmt, pages, H, Dh, seed=3)  # what was there stays where nothing is written
    table = _kv.block_table(rng(4), total, pages)
    dev = c.device(ops)
    k, v = (make_rows(oracle, int(offs[-1]), H * Dh, dtype, 10 + i) for i in range(2))
    if len(k) > 2:
        k[1] = 0  # a row of zeros: scale 1
    tabs = [ops.dev(a) for a in (offs, np.array(start, np.int32), table)]
    ops.kv_write(dev, ops.dev(k), ops.dev(v), *tabs)
    expect_write(oracle, c, k, v, offs, start, table)
    same(ops, dev, c)
    for bf16 in (True, False):
        got = ops.kv_read(dev, *tabs, len(k), bf16=bf16)
        for which, g in zip("kv", got):
            want = np.zeros((len(k), H, Dh), np.float32)
            for s in range(len(start)):
                for i in range(offs[s], offs[s + 1]):
                    page, t = c.find(table, s, start[s] + i - int(offs[s]))
                    for h in range(H):
                        # the product of a code and an fp32 scale, rounded to fp32
                        want[i, h] = c.token(page, h, t)["kv".index(which)].astype(np.float32)
            g = ops.host(g, np.uint16) if bf16 else ops.host(g)
            assert np.array_equal(g, D.to_bf16_bits(oracle, want).reshape(g.shape) if bf16 else want), which


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_write_accepted_rows_of_strided_slices(oracle, ops, fmt):
    """Keys and values as slices of one fused projection at an odd element
    offset (no vector loads), the accepted rows named by an index with entries
    outside the rows."""
    H, Dh, n = 2, 80, 24
    x = make_rows(oracle, n, 401, "bf16", 5)
    t = ops.dev(x)
    new, start = [3, 0, 4], [62, 9, 0]
    rows = np.array([1, 5, -1, 8, 9, 24, 23], np.int32)
    offs, total = offsets_of(new), [a + b for a, b in zip(new, start)]
    c = _kv.HostCache(fmt, 6, H, Dh, seed=8)
    table = _kv.block_table(rng(1), total, 6)
    dev = c.device(ops)
    ops.kv_write(dev, t[:, 1:161], t[:, 241:401], ops.dev(offs), ops.dev(np.array(start, np.int32)), ops.dev(table),
                 rows=ops.dev(rows))
    expect_write(oracle, c, x[:, 1:161], x[:, 241:401], offs, start, table, rows)
    same(ops, dev, c)


def test_missing_pages_are_skipped_and_read_as_zeros(oracle, ops):
    """Entries outside the cache's pages, positions past the table and before
    zero, offsets outside the rows: nothing else is touched."""
    H, Dh = 2, 64
    c = _kv.HostCache("int8", 5, H, Dh, seed=2)
    table = np.array([[0, 5, 2], [-1, 1, 3], [4, -2147483648, 2147483647]], np.int32)
    start = np.array([10, 60, 150], np.int32)
    new = [200, 70, 60]
    offs = offsets_of(new)
    k, v = (make_rows(oracle, 330, H * Dh, "f32", 20 + i) for i in range(2))
    dev = c.device(ops)
    tabs = [ops.dev(a) for a in (offs, start, table)]
    ops.kv_write(dev, ops.dev(k), ops.dev(v), *tabs)
    expect_write(oracle, c, k, v, offs, start, table)
    same(ops, dev, c)
    got = [ops.host(x) for x in ops.kv_read(dev, *tabs, 330, bf16=False)]
    for s in range(3):
        for i in range(offs[s], offs[s + 1]):
            at = c.find(table, s, int(start[s]) + i - int(offs[s]))
            for h in range(H):
                want = (np.zeros(Dh), np.zeros(Dh)) if at is None else c.token(at[0], h, at[1])
                assert np.array_equal(got[0][i, h], want[0].astype(np.float32))
                assert np.array_equal(got[1][i, h], want[1].astype(np.float32))
    # negative positions and offsets outside [0, rows]: clamped, dropped
    before = {n: ops.host(getattr(dev, n)).copy() for n in ("k", "v", "k_scales", "v_scales")}
    ops.kv_write(dev, ops.dev(k), ops.dev(v), ops.dev(np.array([-5, -1, 400, 900], np.int32)),
                 ops.dev(np.array([-1000, -2000, 500], np.int32)), tabs[2])
    for n, b in before.items():
        assert np.array_equal(ops.host(getattr(dev, n)), b), n
    out = ops.kv_read(dev, ops.dev(np.array([-5, -1, 400, 900], np.int32)),
                      ops.dev(np.array([-1000, -2000, 500], np.int32)), tabs[2], 330, bf16=False)
    assert not ops.host(out[0]).any() and not ops.host(out[1]).any()


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_write_nan_and_extreme_rows(oracle, ops, fmt):
    """NaN never wins a row's maximum; subnormal and huge rows keep the rule."""
    H, Dh = 1, 32
    k = rng(9).standard_normal((6, Dh)).astype(np.float32)
    k[0, 3] = np.nan
    k[1] = np.nan
    k[2] *= 1e-42
    k[3] *= 1e37
    k[4] = 0
    k[4, 7] = -0.0
    c = _kv.HostCache(fmt, 1, H, Dh)
    dev = c.device(ops)
    offs, start, table = np.array([0, 6], np.int32), np.array([30], np.int32), np.array([[0]], np.int32)
    ops.kv_write(dev, ops.dev(k), ops.dev(k), *[ops.dev(a) for a in (offs, start, table)])
    expect_write(oracle, c, k, k, offs, start, table)
    same(ops, dev, c)


# ---- attention --------------------------------------------------------------

def bits(oracle, x):
    return D.to_bf16_bits(oracle, np.ascontiguousarray(x, np.float32)).reshape(x.shape)


def tree_masks(g, n, chain=False):
    words = []
    for T in n:
        tree = []
        for i in range(T):
            parent = -1 if i == 0 else i - 1 if chain else int(g.integers(-1, i))
            tree.append((tree[parent] if parent >= 0 else 0) | 1 << i)
        words += tree
    return np.array(words, np.uint64)


class Case:
    """Inputs of one attention call, on the host and on the GPU."""

    def __init__(self, oracle, ops, fmt, Hq, H, Dh, lengths, new, seed=0, tree=True, sharp=2.0, spare=2, width=None):
        g = rng(seed)
        self.oracle, self.ops, self.new = oracle, ops, new
        pages = sum(-(-n // 64) for n in lengths) + spare
        self.c = _kv.HostCache(fmt, pages, H, Dh, seed=seed + 1)
        self.table = _kv.block_table(g, lengths, pages, width)
        self.offs, self.lengths = offsets_of(new), np.array(lengths, np.int32)
        n = int(self.offs[-1])
        self.q = bits(oracle, g.standard_normal((n, Hq, Dh)) * sharp)
        self.k, self.v = (bits(oracle, g.standard_normal((n, H, Dh))) for _ in range(2))
        self.tree = tree_masks(g, new) if tree else None
        self.scale = float(np.float32(Dh ** -0.5))

    def run(self, max_new=None, workspace=True, new=True, out=None):
        ops = self.ops
        dev = self.c.device(ops)
        n, Hq, _ = self.q.shape
        max_new = max(self.new + [0]) if max_new is None else max_new
        ws = ops.kv_attn_workspace(dev, len(self.new), n, max_new, self.table.shape[1], Hq) if workspace else None
        return ops.kv_attn(dev, ops.dev(self.q), ops.dev(self.offs), ops.dev(self.lengths), ops.dev(self.table),
                           ops.dev(self.k) if new else None, ops.dev(self.v) if new else None,
                           tree=None if self.tree is None else ops.dev(self.tree.view(np.int64)), scale=self.scale,
                           max_new=max_new, workspace=ws, out=out)

    def want(self, new=True):
        f = D.bf16_bits_to_f32
        return _kv.attention(self.c, f(self.q), self.offs, self.lengths, self.table, f(self.k) if new else None,
                             f(self.v) if new else None, self.tree, self.scale)

    def check(self, **kw):
        want, bound = self.want(new=kw.get("new", True))
        got = D.bf16_bits_to_f32(self.ops.host(self.run(**kw), np.uint16))
        assert np.isfinite(got).all()
        off = np.abs(got - want)
        assert (off <= bound).all(), f"worst {np.max(off / np.maximum(bound, 1e-300)):.2f} of the bound"


@pytest.mark.parametrize("Hq,H,Dh", [(8, 2, 128), (4, 4, 64), (6, 2, 96), (15, 5, 80), (16, 1, 128), (3, 3, 256), (2, 1, 40),
                                     (4, 2, 192), (5, 1, 75), (32, 2, 64)])
@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_decode(oracle, ops, fmt, Hq, H, Dh):
    Case(oracle, ops, fmt, Hq, H, Dh, [0, 1, 63, 64, 65, 200, 517], [1] * 7, seed=Dh).check()


@pytest.mark.parametrize("T", [2, 3, 5, 16, 17, 33, 63, 64])
@pytest.mark.parametrize("fmt,Hq,H,Dh", [("int8", 8, 2, 128), ("fp8", 3, 1, 64), ("fp8", 2, 2, 256), ("int8", 10, 2, 96)])
def test_trees(oracle, ops, fmt, Hq, H, Dh, T):
    Case(oracle, ops, fmt, Hq, H, Dh, [130, 0, 64], [T, T, max(1, T // 2)], seed=T).check()


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_ragged_trees_and_empty_sequences(oracle, ops, fmt):
    """Sequences without new tokens, without cached ones, without either."""
    Case(oracle, ops, fmt, 8, 2, 128, [100, 0, 0, 300, 64, 1], [5, 0, 3, 1, 0, 40], seed=3).check()


def test_many_sequences(oracle, ops):
    """More sequences than one step of the tile list's scan."""
    g = rng(6)
    lengths = [int(x) for x in g.integers(0, 150, 150)]
    Case(oracle, ops, "fp8", 2, 1, 64, lengths, [int(x) for x in g.integers(0, 3, 150)], seed=8).check()


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("workspace", [True, False])
def test_long_context_splits(oracle, ops, fmt, workspace):
    Case(oracle, ops, fmt, 4, 1, 64, [9001, 40], [1, 2], seed=4).check(workspace=workspace)
    Case(oracle, ops, fmt, 6, 2, 128, [4097], [9], seed=5).check(workspace=workspace)


def test_causal_chain_without_masks(oracle, ops):
    """tree = NULL is the chain, whatever the chain's length."""
    Case(oracle, ops, "int8", 4, 2, 64, [70, 0], [64, 7], seed=2, tree=False).check()


def test_cache_only(oracle, ops):
    """No new keys: every query sees the cached tokens, those of an empty
    sequence nothing."""
    c = Case(oracle, ops, "fp8", 8, 2, 128, [100, 0, 64], [3, 2, 1], seed=2)
    c.check(new=False)
    got = c.ops.host(c.run(new=False), np.uint16)
    assert not got[3:5].any()


def test_rows_that_see_nothing(oracle, ops):
    """Empty masks over an empty cache, and masks whose only bits are past the
    sequence's tokens: zeros; with cached tokens: those alone."""
    c = Case(oracle, ops, "int8", 8, 2, 64, [0, 90], [4, 4], seed=2)
    c.tree = np.array([0, 1, 1 << 63, 0b0110, 0, 0b1000, 1 << 40, 0b1111], np.uint64)
    c.check()
    got = c.ops.host(c.run(), np.uint16)
    assert not got[0].any() and not got[2].any() and got[1].any()


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_garbage_past_the_end_and_in_masked_places(oracle, ops, fmt):
    """NaN and infinite scales and codes past a sequence's length, and in the
    new tokens that a row does not see, change nothing."""
    c = Case(oracle, ops, fmt, 8, 2, 128, [70, 129, 0], [3, 2, 2], seed=7)
    clean = c.ops.host(c.run(), np.uint16).copy()
    for s in range(3):
        L = int(c.lengths[s])
        if L % 64:
            page = c.table[s, L // 64]
            t = np.arange(L % 64, 64)
            c.c.ks[page][:, t] = np.array([np.nan, np.inf, -np.inf, 3e38], np.float32)[t % 4]
            c.c.vs[page][:, t] = np.array([np.inf, np.nan, 3e38, -np.inf], np.float32)[t % 4]
            if fmt == "fp8":
                c.c.k[page][:, t] = 0x7f
                c.c.v[page][:, :, _kv.SLOTS[t]] = 0xff
    assert np.array_equal(c.ops.host(c.run(), np.uint16), clean)
    # the last new token of each sequence is seen by itself alone
    last = c.offs[1:] - 1
    c.tree = np.array([0b001, 0b011, 0b100, 0b01, 0b10, 0b01, 0b10], np.uint64)
    clean = c.ops.host(c.run(), np.uint16).copy()
    others = np.setdiff1d(np.arange(7), last)
    for kbad, vbad in ((0x7fc0, 0x3f80), (0x3f80, 0x7fc0), (0x7f80, 0xff80)):
        c.k[last], c.v[last] = kbad, vbad
        got = c.ops.host(c.run(), np.uint16)
        assert np.array_equal(got[others], clean[others])
    assert not np.isfinite(D.bf16_bits_to_f32(got[last])).any()


def test_missing_pages_are_not_seen(oracle, ops):
    c = Case(oracle, ops, "int8", 4, 2, 64, [300, 200, 64], [2, 1, 1], seed=9)
    c.table[0, 1], c.table[0, 4], c.table[1, 0], c.table[2, 0] = -1, c.c.pages, 2147483647, -2147483648
    c.check()


def test_lengths_outside_the_table(oracle, ops):
    """Lengths are clamped to [0, 64 * max_pages]."""
    c = Case(oracle, ops, "int8", 4, 2, 64, [128, 100], [1, 1], seed=9)
    c.lengths[:] = [128, 128]
    c.table[1] = c.table[0]
    want = c.ops.host(c.run(), np.uint16).copy()
    c.lengths[:] = [2147483647, 4000]
    assert np.array_equal(c.ops.host(c.run(), np.uint16), want)
    c.lengths[:] = [0, 0]
    want = c.ops.host(c.run(), np.uint16).copy()
    c.lengths[:] = [-5, -2147483648]
    assert np.array_equal(c.ops.host(c.run(), np.uint16), want)


def test_tokens_past_max_new_are_left_alone(oracle, ops):
    c = Case(oracle, ops, "int8", 4, 2, 64, [100, 30], [5, 2], seed=3, tree=False)
    want = c.ops.host(c.run(), np.uint16).copy()
    out = c.ops.empty(c.q.shape, np.int16)
    out.fill_(77)
    got = c.ops.host(c.run(max_new=2, out=out), np.uint16)
    assert np.array_equal(got[:2], want[:2]) and np.array_equal(got[5:], want[5:]) and (got[2:5] == 77).all()


def test_sharp_and_flat_softmax(oracle, ops):
    """Scores in the hundreds (one weight is everything) and all equal."""
    for sharp in (60.0, 0.0):
        Case(oracle, ops, "int8", 8, 2, 128, [700, 64], [3, 1], seed=12, sharp=sharp).check()


def test_value_scales_far_apart(oracle, ops):
    """Tokens whose values are 10^4 times the others', and zero scales."""
    c = Case(oracle, ops, "int8", 8, 2, 64, [200, 130], [2, 2], seed=13)
    c.c.vs[:, :, ::7] *= 1e4
    c.c.vs[:, :, 3::11] = 0
    c.c.ks[:, :, 5::13] = 0
    c.check()


def test_strides_alignment_and_other_stream(oracle, ops):
    """q, k and v as slices of one projection at an odd offset, on a stream
    that is not the default one."""
    import torch
    c = Case(oracle, ops, "fp8", 8, 2, 64, [200, 0, 65], [3, 1, 2], seed=14)
    n = len(c.q)
    want = c.ops.host(c.run(), np.uint16).copy()
    x = np.zeros((n, 777), np.uint16)
    x[:, 1:513], x[:, 513:641], x[:, 643:771] = (a.reshape(n, -1) for a in (c.q, c.k, c.v))
    side = torch.cuda.Stream()
    t, dev = ops.dev(x), c.c.device(ops)
    tabs = [ops.dev(a) for a in (c.offs, c.lengths, c.table)]
    tree = ops.dev(c.tree.view(np.int64))
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ws = ops.kv_attn_workspace(dev, 3, n, 3, c.table.shape[1], 8)
        got = ops.kv_attn(dev, t[:, 1:513], *tabs, t[:, 513:641], t[:, 643:771], tree=tree, max_new=3, workspace=ws)
    side.synchronize()
    assert np.array_equal(ops.host(got, np.uint16), want)


def test_repeats_are_bit_equal(oracle, ops):
    c = Case(oracle, ops, "int8", 8, 2, 128, [3000, 900, 10], [4, 4, 4], seed=15)
    first = c.ops.host(c.run(), np.uint16).copy()
    for _ in range(3):
        assert np.array_equal(c.ops.host(c.run(), np.uint16), first)


def test_decode_step_in_a_graph(oracle, ops):
    """Write, attend and read back captured once; replays with other inputs and
    lengths equal the eager calls on those."""
    import torch
    c = Case(oracle, ops, "int8", 8, 2, 128, [64, 700, 0], [1, 2, 1], seed=16, width=12)
    big = _kv.HostCache("int8", 36, 2, 128, seed=5)  # every sequence has 12 pages, filled or not
    c.table[:] = rng(3).permutation(36).reshape(3, 12)
    dev = big.device(ops)
    n = len(c.q)
    q, k, v = ops.dev(c.q), ops.dev(c.k), ops.dev(c.v)
    offs, lengths, table = ops.dev(c.offs), ops.dev(c.lengths), ops.dev(c.table)
    ws = ops.kv_attn_workspace(dev, 3, n, 2, 12, 8)
    out = ops.empty((n, 8, 128), np.int16)
    back = (ops.empty((n, 2, 128), np.int16), ops.empty((n, 2, 128), np.int16))

    def step():
        ops.kv_attn(dev, q, offs, lengths, table, k, v, max_new=2, workspace=ws, out=out)
        ops.kv_write(dev, k, v, offs, lengths, table)
        ops.kv_read(dev, offs, lengths, table, n, out=back)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for rep in range(4):
        q.copy_(ops.dev(bits(oracle, rng(50 + rep).standard_normal(c.q.shape) * 2)))
        k.copy_(ops.dev(bits(oracle, rng(60 + rep).standard_normal(c.k.shape))))
        lengths.copy_(ops.dev(np.array([64 + rep, 700 - 60 * rep, rep], np.int32)))
        step()
        want = [ops.host(t, np.uint16).copy() for t in (out, *back)]
        for t in (out, *back):
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for t, w in zip((out, *back), want):
            assert np.array_equal(ops.host(t, np.uint16), w), rep


def test_offsets_past_32_bits(oracle, ops):
    """The last pages of a cache of over 4 GiB of codes for keys and values
    each."""
    import torch
    H, Dh = 16, 256
    page_bytes = H * 64 * Dh
    pages = (1 << 32) // page_bytes + 40
    dev = ops.KvCache("fp8", pages, H, Dh, *(torch.zeros(pages * page_bytes, dtype=torch.uint8, device="cuda")
                                             for _ in range(2)),
                      *(torch.zeros(pages * H * 64, dtype=torch.float32, device="cuda") for _ in range(2)))
    g = rng(1)
    new, start = [100, 3], [30, 64]
    offs, total = offsets_of(new), [130, 67]
    # a small host cache stands for the pages that are used; ids are shifted by where they lie
    small = _kv.HostCache("fp8", 5, H, Dh)
    table = _kv.block_table(g, total, 5)
    k, v = (make_rows(oracle, 103, H * Dh, "bf16", 70 + i) for i in range(2))
    shifted = ops.dev(np.where(table >= 0, table + pages - 5, table).astype(np.int32))
    tabs = [ops.dev(offs), ops.dev(np.array(start, np.int32)), shifted]
    ops.kv_write(dev, ops.dev(k), ops.dev(v), *tabs)
    expect_write(oracle, small, k, v, offs, start, table)
    tail = 5 * page_bytes
    assert np.array_equal(ops.host(dev.k[-tail:]), small.k.reshape(-1))
    assert np.array_equal(ops.host(dev.v[-tail:]), small.v.reshape(-1))
    assert not bool(dev.k[:-tail].any()) and not bool(dev.v[:-tail].any())
    back = ops.kv_read(dev, *tabs, 103, bf16=False)
    page, t = small.find(table, 0, 129)
    assert np.array_equal(ops.host(back[1][99, 7]), small.token(page, 7, t)[1].astype(np.float32))
    c = Case(oracle, ops, "fp8", 16, H, Dh, total, [1, 1], seed=21)
    c.c, c.table = small, table
    want, bound = c.want()
    got = ops.kv_attn(dev, ops.dev(c.q), ops.dev(c.offs), ops.dev(c.lengths), shifted, ops.dev(c.k), ops.dev(c.v),
                      tree=ops.dev(c.tree.view(np.int64)), scale=c.scale)
    assert (np.abs(D.bf16_bits_to_f32(ops.host(got, np.uint16)) - want) <= bound).all()
    del dev
    torch.cuda.empty_cache()
