"""Attention over the 8-bit cache at the sizes where its kernel changes form:
head sizes of every operand width, query blocks of more than one tile, more
pages a wave than one read of the block table, splits joined over little and
much workspace, running maxima and value exponents that keep moving.  Against
64-bit numpy (tests/_kv.py)."""
import numpy as np
import pytest

from tests import _data as D
from tests import _kv
from tests.test_kv_gpu import Case, expect_write, make_rows, offsets_of, rng, same

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(lib):
    from longhornai_amd import ops as _ops
    return _ops


@pytest.mark.parametrize("Dh", [1, 2, 7, 8, 9, 31, 33, 63, 97, 129, 160, 193, 224, 255])
@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_head_sizes(oracle, ops, fmt, Dh):
    """One tile of queries and several, every operand width, odd row lengths."""
    Case(oracle, ops, fmt, 6, 2, Dh, [70, 0, 200], [1, 1, 1], seed=Dh).check()
    Case(oracle, ops, fmt, 6, 2, Dh, [70, 0, 129], [11, 7, 17], seed=Dh + 1).check()


@pytest.mark.parametrize("Hq,H,T", [(48, 2, 3), (34, 2, 1), (70, 1, 1), (33, 1, 2), (64, 4, 64), (7, 7, 33)])
def test_query_blocks(oracle, ops, Hq, H, T):
    """Groups that do not divide a tile, tokens cut by the end of a block."""
    Case(oracle, ops, "int8", Hq, H, 32, [150, 64], [T, max(1, T - 1)], seed=Hq + T).check()


@pytest.mark.parametrize("workspace", [True, False])
def test_more_pages_a_wave_than_a_read_of_the_table(oracle, ops, workspace):
    """40000 tokens: 625 pages over at most eight waves without a workspace."""
    c = Case(oracle, ops, "fp8", 1, 1, 32, [40000], [1], seed=3, spare=9)
    c.table[0, 130], c.table[0, 517], c.table[0, 518] = -1, c.c.pages, -7
    c.check(workspace=workspace)


@pytest.mark.parametrize("part", [0, 1, 16, 4000, 0.1, 0.34, 0.6, 1.0])
def test_workspace_of_any_size(oracle, ops, part):
    """A smaller workspace means fewer splits, never another answer."""
    import torch
    c = Case(oracle, ops, "int8", 8, 2, 64, [4500, 900, 0, 2300], [2, 1, 1, 3], seed=5)
    dev = c.c.device(ops)
    full = ops.kv_attn_workspace(dev, 4, len(c.q), 3, c.table.shape[1], 8)
    assert full is not None
    size = int(part * full.numel()) if isinstance(part, float) else part
    guard = torch.full((size + 64,), 77, dtype=torch.uint8, device="cuda")
    got = ops.kv_attn(dev, ops.dev(c.q), ops.dev(c.offs), ops.dev(c.lengths), ops.dev(c.table), ops.dev(c.k),
                      ops.dev(c.v), tree=ops.dev(c.tree.view(np.int64)), scale=c.scale, max_new=3,
                      workspace=guard[:size] if size else None)
    want, bound = c.want()
    assert (np.abs(D.bf16_bits_to_f32(ops.host(got, np.uint16)) - want) <= bound).all()
    assert bool((guard[size:] == 77).all())


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("rise", [1.6, 1 / 1.6])
def test_maxima_and_value_scales_that_keep_moving(oracle, ops, fmt, rise):
    """Scores and value scales that grow (or shrink) from page to page, so the
    running maximum and the running exponent change at each."""
    c = Case(oracle, ops, fmt, 8, 2, 64, [1500, 700], [3, 9], seed=6)
    for s in range(2):
        for i, page in enumerate(c.table[s]):
            if page >= 0:
                c.c.ks[page] *= np.float32(rise ** (i / 2))
                c.c.vs[page] *= np.float32(rise ** (2 * i))
    c.check()


def test_equal_scores_far_from_zero(oracle, ops):
    """Every score the same large number of either sign: plain means."""
    for sign in (1.0, -1.0):
        c = Case(oracle, ops, "int8", 4, 1, 32, [900], [2], seed=8)
        c.c.k[...] = 0
        c.c.k[..., 0] = 127
        c.c.ks[...] = 1.0
        c.q[...] = 0
        c.q[..., 0] = D.to_bf16_bits(oracle, np.array([sign * 8.0], np.float32))[0]
        c.k[...] = 0
        c.k[..., 0] = D.to_bf16_bits(oracle, np.array([127.0], np.float32))[0]
        c.check()


def test_missing_pages_ahead_of_far_scores(oracle, ops):
    """Waves whose first pages are missing, then scores of -180 alone."""
    c = Case(oracle, ops, "int8", 4, 1, 32, [2500], [2], seed=8)
    c.c.k[...] = 0
    c.c.k[..., 0] = 127
    c.c.ks[...] = 1.0
    c.q[...] = 0
    c.q[..., 0] = D.to_bf16_bits(oracle, np.array([-8.0], np.float32))[0]
    c.k[...] = 0
    c.k[..., 0] = D.to_bf16_bits(oracle, np.array([127.0], np.float32))[0]
    for gone in (range(0, 9), range(0, 39), range(0, 40)):
        table = c.table.copy()
        c.table[0, list(gone)] = -1
        c.check()
        c.check(new=False) if len(gone) < 40 else None
        c.table = table


@pytest.mark.parametrize("T", [1, 3, 40, 64])
@pytest.mark.parametrize("Hq,Dh", [(1, 32), (4, 128), (3, 256)])
def test_far_scores_of_queries_that_see_none_of_a_waves_new_tokens(oracle, ops, Hq, Dh, T):
    """Every score -180 or 180.  Queries that see new tokens share waves with
    some that see none of them, or none of the 32 that the wave has."""
    for q in (-8.0, 8.0):
        c = Case(oracle, ops, "int8", Hq, 1, Dh, [130, 700, 0], [T, T, T], seed=T)
        c.scale = float(np.float32(32 ** -0.5))
        c.c.k[...] = 0
        c.c.k[..., 0] = 127
        c.c.ks[...] = 1.0
        c.q[...] = 0
        c.q[..., 0] = D.to_bf16_bits(oracle, np.array([q], np.float32))[0]
        c.k[...] = 0
        c.k[..., 0] = D.to_bf16_bits(oracle, np.array([127.0], np.float32))[0]
        c.check()
        c.tree[:] = [(1 << (i % T + 1)) - 1 for i in range(3 * T)]
        c.check()
        c.tree[::2] = 0
        c.check()


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_nan_stays_with_the_queries_that_see_it(oracle, ops, fmt):
    """A NaN key scale, a NaN value scale and (fp8) a NaN code of tokens that
    are seen reach their own sequence and kv head alone."""
    c = Case(oracle, ops, fmt, 8, 2, 64, [100, 200, 64], [2, 2, 1], seed=9)
    clean = c.ops.host(c.run(), np.uint16).copy()
    c.c.ks[c.table[0, 0], 0, 5] = np.nan
    c.c.vs[c.table[1, 2], 1, 3] = np.nan
    if fmt == "fp8":
        c.c.v[c.table[2, 0], 0, 7, _kv.slot(9)] = 0x7f
    got = c.ops.host(c.run(), np.uint16)
    nan = np.isnan(D.bf16_bits_to_f32(got))
    hit = np.zeros_like(nan)
    hit[0:2, :4] = True
    hit[2:4, 4:] = True
    if fmt == "fp8":
        hit[4, :4, 7] = True
    assert (nan == hit).all()
    assert np.array_equal(got[~hit], clean[~hit])


def test_results_at_an_odd_address(oracle, ops):
    """Rows of results that allow no wide stores."""
    import torch
    c = Case(oracle, ops, "int8", 4, 2, 64, [2000, 70], [1, 2], seed=10)
    want = c.ops.host(c.run(), np.uint16).copy()
    n = want.size
    buf = torch.full((n + 2,), 99, dtype=torch.int16, device="cuda")
    c.run(out=buf[1:n + 1].view(want.shape))
    got = c.ops.host(buf, np.uint16)
    assert got[0] == 99 and got[-1] == 99 and np.array_equal(got[1:-1].reshape(want.shape), want)


def test_split_decode_in_a_graph(oracle, ops):
    """Lengths that change between replays, from one split to many and back."""
    import torch
    c = Case(oracle, ops, "int8", 8, 2, 64, [6000, 100], [1, 1], seed=11)
    c.table[1, :] = c.table[0, :]  # (shared pages: neither sequence writes)
    dev, n = c.c.device(ops), len(c.q)
    q, k, v = ops.dev(c.q), ops.dev(c.k), ops.dev(c.v)
    offs, lengths, table = ops.dev(c.offs), ops.dev(c.lengths), ops.dev(c.table)
    ws = ops.kv_attn_workspace(dev, 2, n, 1, c.table.shape[1], 8)
    assert ws is not None
    out = ops.empty((n, 8, 64), np.int16)

    def step():
        ops.kv_attn(dev, q, offs, lengths, table, k, v, max_new=1, workspace=ws, out=out)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for pair in ((6000, 100), (1, 6000), (0, 0), (6000, 5999), (64, 3000)):
        lengths.copy_(ops.dev(np.array(pair, np.int32)))
        step()
        want = ops.host(out, np.uint16).copy()
        c.lengths[:] = pair
        c.tree = None
        oracle_want, bound = c.want()
        assert (np.abs(D.bf16_bits_to_f32(want) - oracle_want) <= bound).all(), pair
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(ops.host(out, np.uint16), want), pair


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("Dh,dtype", [(64, "bf16"), (128, "f32"), (250, "bf16"), (3, "f32")])
def test_write_rows_of_every_size(oracle, ops, fmt, Dh, dtype):
    """Rows from 2^-149 to 2^127 beside each other, of zeros of either sign and
    of values on both sides of the smallest e4m3 step: the plain way and the
    way with the edge cases meet in one workgroup."""
    H, n = 2, 80
    g = rng(3)
    k = (g.standard_normal((n, H * Dh)) * np.exp2(g.integers(-20, 20, (n, 1)))).astype(np.float32)
    k[5] *= np.float32(2.0 ** 100)
    k[6] = 2.0 ** -149
    k[7] = g.standard_normal(H * Dh) * 2.0 ** -120
    k[8] = -0.0
    k[9, ::3] = 3e38
    k[10, 1::4] = np.nan
    x = np.array([448.0] + [2.0 ** -9 * f for f in (1.0, 0.999, 0.75, 0.5, 0.501, 1.001, -0.6, -0.4)], np.float32)
    k[11] = np.resize(x, H * Dh)
    v = k[::-1].copy()
    if dtype == "bf16":
        k, v = D.to_bf16_bits(oracle, k), D.to_bf16_bits(oracle, v)
    c = _kv.HostCache(fmt, 3, H, Dh, seed=4)
    table, offs, start = np.array([[2, 0]], np.int32), offsets_of([n]), np.array([40], np.int32)
    dev = c.device(ops)
    with np.errstate(all="ignore"):
        ops.kv_write(dev, ops.dev(k), ops.dev(v), *[ops.dev(a) for a in (offs, start, table)])
        expect_write(oracle, c, k, v, offs, start, table)
    same(ops, dev, c)


def test_read_of_single_tokens(oracle, ops):
    """One token at each place of a page: its own row and nothing else."""
    c = _kv.HostCache("int8", 3, 2, 96, seed=5)
    dev = c.device(ops)
    table = np.array([[1, 2]] * 128, np.int32)
    start = np.arange(128, dtype=np.int32)
    k, v = ops.kv_read(dev, ops.dev(offsets_of([1] * 128)), ops.dev(start), ops.dev(table), 128, bf16=False)
    k, v = ops.host(k), ops.host(v)
    for i in range(128):
        for h in range(2):
            a, b = c.token(1 + i // 64, h, i % 64)
            assert np.array_equal(k[i, h], a.astype(np.float32)) and np.array_equal(v[i, h], b.astype(np.float32))


def test_rows_made_for_both_ways(oracle, ops):
    """make_rows' values through one page in two calls equal one call."""
    x = make_rows(oracle, 64, 2 * 128, "bf16", 77)
    caches = []
    for parts in ((64,), (1, 30, 33)):
        c = _kv.HostCache("fp8", 1, 2, 128)
        dev, at = c.device(ops), 0
        for n in parts:
            ops.kv_write(dev, ops.dev(x[at:at + n]), ops.dev(x[at:at + n]), ops.dev(offsets_of([n])),
                         ops.dev(np.array([at], np.int32)), ops.dev(np.array([[0]], np.int32)))
            at += n
        caches.append([ops.host(t).copy() for t in (dev.k, dev.v, dev.k_scales, dev.v_scales)])
    for a, b in zip(*caches):
        assert np.array_equal(a, b)
