"""Attention of prompts and chunks on the GPU against 64-bit numpy, with bounds
derived in tests/_prefill.py."""
import numpy as np
import pytest

from tests import _data as D
from tests import _kv
from tests._prefill import Case, check

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(lib):
    from longhornai_amd import ops as _ops
    return _ops


def f32(ops, t):
    return D.bf16_bits_to_f32(ops.host(t, np.uint16))


# (query heads, kv heads, head_dim, new tokens of each sequence)
PROMPTS = [
    (1, 1, 1, [3]), (1, 1, 5, [70]), (2, 1, 8, [1, 2, 65]), (4, 2, 32, [64]), (4, 4, 33, [130]),
    (15, 5, 80, [40, 0, 129]), (8, 2, 64, [63, 1, 64, 0, 65]), (3, 1, 96, [200]), (8, 2, 128, [257, 31]),
    (8, 1, 128, [33, 300]), (2, 2, 160, [100]), (6, 2, 192, [90]), (2, 1, 200, [129]), (4, 2, 224, [70]),
    (4, 1, 256, [150, 2]), (2, 2, 255, [66]), (7, 1, 75, [97]), (32, 8, 128, [1]), (16, 1, 64, [16, 17]),
]


@pytest.mark.parametrize("Hq,H,dim,new", PROMPTS)
def test_prompts(oracle, ops, Hq, H, dim, new):
    c = Case(oracle, None, Hq, H, dim, [0] * len(new), new, seed=dim + Hq)
    check(f32(ops, c.run(ops)), *c.want())


# lengths: none, one, inside a page, its end, past it
CHUNKS = [
    (4, 2, 64, [0, 1, 63, 64, 65], [5, 1, 70, 0, 64]), (8, 2, 128, [300, 0, 129], [130, 65, 1]),
    (15, 5, 80, [100, 7], [33, 90]), (1, 1, 1, [70], [3]), (2, 1, 33, [64, 200], [66, 2]), (3, 3, 96, [90], [70]),
    (4, 1, 160, [130], [65]), (2, 2, 192, [200], [64]), (4, 2, 224, [65], [40]), (4, 1, 256, [190, 0], [100, 3]),
    (8, 1, 255, [64], [9]), (64, 8, 128, [128], [5]), (16, 2, 40, [1000], [12]),
]


@pytest.mark.parametrize("Hq,H,dim,lengths,new", CHUNKS)
@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_chunks(oracle, ops, fmt, Hq, H, dim, lengths, new):
    c = Case(oracle, fmt, Hq, H, dim, lengths, new, seed=dim + Hq)
    check(f32(ops, c.run(ops)), *c.want())


@pytest.mark.parametrize("fmt", [None, "int8"])
@pytest.mark.parametrize("dim,shift", [(64, 0), (64, 8), (64, 1), (80, 4), (75, 3), (5, 1)])
def test_rows_are_slices_of_one_projection(oracle, ops, fmt, dim, shift):
    """Strided rows, at aligned and odd places: the same result to the bit."""
    c = Case(oracle, fmt, 6, 2, dim, [70, 0], [66, 70], seed=dim)
    assert np.array_equal(ops.host(c.run(ops, wide=True, shift=shift)), ops.host(c.run(ops)))


@pytest.mark.parametrize("Hq,H,dim,lengths,new", [
    (4, 1, 64, [9000], [3]), (2, 1, 128, [5000, 70], [130, 1]), (8, 8, 64, [3000, 2000, 0], [5, 1, 40]),
    (3, 1, 256, [2500], [90])])
def test_few_rows_over_many_keys_are_split(oracle, ops, Hq, H, dim, lengths, new):
    c = Case(oracle, "int8", Hq, H, dim, lengths, new, seed=4)
    want, bound = c.want()
    check(f32(ops, c.run(ops)), want, bound)
    check(f32(ops, c.run(ops, workspace=False)), want, bound)


def test_a_long_prompt_of_one_head_is_split(oracle, ops):
    c = Case(oracle, None, 1, 1, 64, [0], [2600], seed=5)
    want, bound = c.want()
    check(f32(ops, c.run(ops)), want, bound)
    check(f32(ops, c.run(ops, workspace=False)), want, bound)


@pytest.mark.parametrize("room", [0, 16, 100000, 400000])
def test_any_workspace_will_do(oracle, ops, room):
    import torch
    c = Case(oracle, "fp8", 4, 2, 64, [4000, 64], [20, 300], seed=6)
    q, k, v = c.args(ops)
    ws = torch.full((room,), 255, dtype=torch.uint8, device="cuda")
    got = ops.kv_prefill(c.c.device(ops), q, ops.dev(c.offs), ops.dev(c.lengths), ops.dev(c.table), k, v, scale=c.scale,
                         workspace=ws)
    check(f32(ops, got), *c.want())


def test_the_same_bits_every_time(oracle, ops):
    c = Case(oracle, "int8", 8, 2, 128, [5000, 100], [70, 200], seed=7)
    first = ops.host(c.run(ops))
    for _ in range(4):
        assert np.array_equal(ops.host(c.run(ops)), first)


def test_only_the_cache_is_seen(oracle, ops):
    c = Case(oracle, "int8", 4, 2, 64, [130, 0, 64], [70, 2, 1], seed=8)
    got = f32(ops, c.run(ops, new_tokens=False))
    check(got, *c.want(new_tokens=False))
    assert not got[70:72].any()  # (nothing to see: zeros)


@pytest.mark.parametrize("new_tokens", [True, False])
def test_missing_pages_are_not_seen(oracle, ops, new_tokens):
    c = Case(oracle, "fp8", 4, 2, 64, [300, 200, 64], [70, 3, 2], seed=9)
    c.table[0, 1], c.table[0, 4], c.table[1, 0], c.table[2, 0] = -1, c.c.pages, 2 ** 31 - 1, -2 ** 31
    got = f32(ops, c.run(ops, new_tokens=new_tokens))
    check(got, *c.want(new_tokens=new_tokens))
    if not new_tokens:
        assert not got[73:].any()


def test_lengths_outside_the_table_are_clamped(oracle, ops):
    c = Case(oracle, "int8", 4, 2, 64, [128, 60], [5, 4], seed=10)
    c.lengths = np.array([100000, -7], np.int32)
    got = f32(ops, c.run(ops))
    c.lengths = np.array([128, 0], np.int32)
    check(got, *c.want())


def test_rows_of_no_sequence_stay(oracle, ops):
    c = Case(oracle, "int8", 4, 2, 64, [70, 10], [66, 70], seed=11, pad=40)
    c.offs = np.array([7, 73, 143], np.int32)
    out = ops.dev(np.full(c.q.shape, 77, np.int16))
    c.run(ops, out=out)
    got = ops.host(out)
    assert (got[:7] == 77).all() and (got[143:] == 77).all()
    want, bound = c.want()
    check(D.bf16_bits_to_f32(got.view(np.uint16)), want, bound, slice(7, 143))
    made = ops.host(c.run(ops))
    assert not made[:7].any() and not made[143:].any() and np.array_equal(made[7:143], got[7:143])


def test_offsets_outside_the_rows_are_clamped(oracle, ops):
    c = Case(oracle, None, 4, 2, 64, [0, 0, 0], [20, 30, 10], seed=12)
    c.offs = np.array([-5, 20, 50, 2 ** 31 - 1], np.int32)
    got = f32(ops, c.run(ops))
    c.offs = np.array([0, 20, 50, 60], np.int32)
    check(got, *c.want())


ODD = [0x7f80, 0xff80, 0x7fc0]  # infinity, -infinity, NaN


@pytest.mark.parametrize("fmt", [None, "int8"])
@pytest.mark.parametrize("aligned", [True, False])
def test_what_a_row_does_not_see_changes_nothing(oracle, ops, fmt, aligned):
    """Infinities, NaN and huge numbers in later tokens, in rows of the next
    sequence and past the last one, in the cache behind a sequence's length: to
    the bit."""
    dim = 64 if aligned else 61
    c = Case(oracle, fmt, 4, 2, dim, [70, 100], [150, 30], seed=13, pad=20)
    clean = ops.host(c.run(ops))
    for t in (100, 120, 149):
        c.k[t], c.v[t] = 0x7fc0, 0x7f80
        c.v[t, 1, :4] = ODD + [0x7f00]
    c.k[180:], c.v[180:], c.q[180:] = 0x7fc0, 0x7fc0, 0x7fc0
    if fmt:  # what the last pages hold behind the tokens
        for s, n in ((0, 70), (1, 100)):
            page = c.table[s, n // 64]
            c.c.ks[page, :, n % 64:], c.c.vs[page, :, n % 64:] = np.nan, np.inf
    got = ops.host(c.run(ops))
    assert np.array_equal(got[:100], clean[:100]) and np.array_equal(got[150:180], clean[150:180])
    # and who sees them has them
    want, bound = c.want()
    assert np.isnan(want[100:150]).all()
    assert np.isnan(D.bf16_bits_to_f32(got.view(np.uint16))[100:150]).all()


def test_e4m3_nan_codes_behind_the_length_are_not_seen(oracle, ops):
    c = Case(oracle, "fp8", 4, 2, 64, [70, 100], [3, 40], seed=14)
    clean = ops.host(c.run(ops))
    for s, n in ((0, 70), (1, 100)):
        page = c.table[s, n // 64]
        c.c.k[page, :, n % 64:] = 0x7f
        c.c.v[page][:, :, _kv.SLOTS[n % 64:]] = 0xff
    assert np.array_equal(ops.host(c.run(ops)), clean)


@pytest.mark.parametrize("value", ODD)
@pytest.mark.parametrize("token", [0, 40, 100])
def test_values_that_are_infinite_or_nan_reach_who_sees_them(oracle, ops, value, token):
    """One channel of one value: that channel of the rows that see it, nothing else."""
    c = Case(oracle, None, 4, 2, 64, [0], [130], seed=15)
    clean = ops.host(c.run(ops))
    c.v[token, 1, 9] = value
    got = ops.host(c.run(ops))
    other = np.ones(got.shape, bool)
    other[token:, 2:, 9] = False
    assert np.array_equal(got[other], clean[other])
    hit = D.bf16_bits_to_f32(got.view(np.uint16))[token:, 2:, 9]
    assert np.isnan(hit).all() if value == 0x7fc0 else (hit == (np.inf if value == 0x7f80 else -np.inf)).all()


def test_scores_of_every_size(oracle, ops):
    """Large queries: one key takes all the weight, the maximum moves often."""
    for gain in (30.0, 1e4, 1e-6):
        c = Case(oracle, "int8", 4, 2, 64, [200], [140], seed=16, gain=gain)
        c.c.ks *= np.linspace(0.2, 3, c.c.ks.size, dtype=np.float32).reshape(c.c.ks.shape)
        check(f32(ops, c.run(ops)), *c.want())


def test_keys_of_minus_infinity_take_no_weight(oracle, ops):
    c = Case(oracle, None, 2, 1, 64, [0], [80], seed=17)
    c.q[..., 0], c.k[10, 0, 0], c.k[70, 0, 0] = 0x3f80, 0xff80, 0xff80
    got, (want, bound) = f32(ops, c.run(ops)), c.want()
    assert np.isfinite(want[:10]).all() and np.isfinite(want[71:]).all()
    check(got, want, bound)


def test_value_scales_of_every_size(oracle, ops):
    c = Case(oracle, "fp8", 4, 2, 64, [300], [20], seed=18)
    c.c.vs *= (2.0 ** np.random.default_rng(1).integers(-60, 60, c.c.vs.shape)).astype(np.float32)
    check(f32(ops, c.run(ops)), *c.want())


def test_agrees_with_attention_of_few_tokens(oracle, ops):
    """kv_attn on the same cache, a chunk of 64: within both roundings."""
    c = Case(oracle, "int8", 8, 2, 128, [300, 64], [64, 20], seed=19)
    a = f32(ops, c.run(ops))
    b = f32(ops, ops.kv_attn(c.c.device(ops), ops.dev(c.q), ops.dev(c.offs), ops.dev(c.lengths), ops.dev(c.table),
                             ops.dev(c.k), ops.dev(c.v), scale=c.scale))
    _, bound = c.want()
    assert (np.abs(a - b) <= 2 * bound).all()


def test_pages_past_4_gib(oracle, ops):
    """Pages whose codes lie past 2^32 bytes: the same bits as in a small cache."""
    import torch
    c = Case(oracle, "int8", 8, 4, 128, [200], [70], seed=20)
    small = ops.host(c.run(ops))
    pages = (1 << 32) // (4 * 64 * 128) + 10
    big = ops.kv_cache("int8", pages, 4, 128)
    ids = pages - 1 - np.arange(c.table.shape[1], dtype=np.int32)[None]
    for p in range(c.table.shape[1]):
        at, to = int(c.table[0, p]), int(ids[0, p])
        for name, src in (("k", c.c.k), ("v", c.c.v), ("k_scales", c.c.ks), ("v_scales", c.c.vs)):
            dst = getattr(big, name)
            dst.view(pages, -1)[to].copy_(ops.dev(src[at].reshape(-1)))
    got = ops.kv_prefill(big, ops.dev(c.q), ops.dev(c.offs), ops.dev(c.lengths), ops.dev(ids), ops.dev(c.k), ops.dev(c.v),
                         scale=c.scale)
    assert np.array_equal(ops.host(got), small)
    del big
    torch.cuda.empty_cache()


def test_many_sequences(oracle, ops):
    """Over 64 of them, of which most have a row or none."""
    g = np.random.default_rng(21)
    new = [int(x) for x in g.integers(0, 4, 150)]
    new[100] = 140
    lengths = [int(x) for x in g.integers(0, 150, 150)]
    c = Case(oracle, "int8", 4, 2, 32, lengths, new, seed=21)
    check(f32(ops, c.run(ops)), *c.want())


# without a cache, where the rows are many: the larger row blocks, at every number of 32 channels
# that has them (the call has the room; most rows are of no sequence)
ROOMY = [
    (32, 8, 128, [300], 4000), (32, 2, 100, [700, 3], 8000), (32, 32, 112, [130], 4000), (32, 4, 97, [65, 0, 70], 13000),
    (16, 4, 256, [150, 600], 4000), (16, 16, 160, [70], 4096), (64, 1, 192, [40], 1100), (16, 2, 224, [129], 4096),
    (32, 4, 255, [33, 90], 2100),
]


@pytest.mark.parametrize("Hq,H,dim,new,pad", ROOMY)
def test_few_rows_in_a_large_call(oracle, ops, Hq, H, dim, new, pad):
    c = Case(oracle, None, Hq, H, dim, [0] * len(new), new, seed=dim, pad=pad)
    n = sum(new)
    want, bound = c.want()
    for workspace in (True, False):
        got = f32(ops, c.run(ops, workspace=workspace))
        check(got, want, bound, slice(0, n))
        assert not got[n:].any()


@pytest.mark.parametrize("dim,shift", [(128, 8), (128, 1), (104, 4), (99, 3)])
def test_slices_of_one_projection_in_a_large_call(oracle, ops, dim, shift):
    c = Case(oracle, None, 32, 8, dim, [0], [200], seed=dim, pad=3900)
    assert np.array_equal(ops.host(c.run(ops, wide=True, shift=shift)), ops.host(c.run(ops)))


@pytest.mark.parametrize("dim", [128, 99])
@pytest.mark.parametrize("value", ODD)
def test_odd_values_in_a_large_call(oracle, ops, dim, value):
    c = Case(oracle, None, 32, 8, dim, [0], [200], seed=dim, pad=3900)
    clean = ops.host(c.run(ops))
    c.v[150, 1, 9] = value
    c.k[200:], c.v[200:], c.q[200:] = 0x7fc0, 0x7fc0, 0x7fc0
    got = ops.host(c.run(ops))
    other = np.ones(got.shape, bool)
    other[150:200, 4:8, 9] = False
    assert np.array_equal(got[other], clean[other])
    assert (got.view(np.uint16)[150:200, 4:8, 9] & 0x7fff >= 0x7f80).all()


def test_a_prompt_of_four_thousand(oracle, ops):
    """Two of the kv heads against 64 bits."""
    from tests._prefill import attention
    c = Case(oracle, None, 32, 8, 128, [0], [4133], seed=30)
    got, f = f32(ops, c.run(ops)), D.bf16_bits_to_f32
    for h in (0, 5):
        q, k, v = f(c.q[:, 4 * h:4 * h + 2]), f(c.k[:, h:h + 1]), f(c.v[:, h:h + 1])
        check(got[:, 4 * h:4 * h + 2], *attention(None, q, c.offs, c.lengths, None, k, v, c.scale))


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_many_sequences_of_which_some_are_split(oracle, ops, fmt):
    g = np.random.default_rng(31)
    new = [int(x) for x in g.integers(0, 3, 140)]
    lengths = [int(x) for x in g.integers(0, 150, 140)]
    for s, n, t in ((3, 3000, 2), (70, 1, 40), (71, 2000, 1), (139, 2500, 9)):
        lengths[s], new[s] = n, t
    c = Case(oracle, fmt, 4, 2, 64, lengths, new, seed=31)
    want, bound = c.want()
    check(f32(ops, c.run(ops)), want, bound)
    check(f32(ops, c.run(ops, workspace=False)), want, bound)


@pytest.mark.parametrize("value", ODD)
@pytest.mark.parametrize("gain", [1.0, 1e4])
def test_odd_values_in_a_split_part_reach_who_sees_them(oracle, ops, gain, value):
    """Whatever its part weighs beside the others (with large queries: nothing)."""
    c = Case(oracle, "int8", 4, 2, 64, [3000], [20], seed=32, gain=gain)
    clean = ops.host(c.run(ops))
    c.v[7, 1, 9] = value
    got = ops.host(c.run(ops))
    other = np.ones(got.shape, bool)
    other[7:, 2:, 9] = False
    assert np.array_equal(got[other], clean[other])
    hit = D.bf16_bits_to_f32(got.view(np.uint16))[7:, 2:, 9]
    assert np.isnan(hit).all() if value == 0x7fc0 else (hit == (np.inf if value == 0x7f80 else -np.inf)).all()


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_sequences_that_share_pages(oracle, ops, fmt):
    """A common prefix held once: the bits of a sequence that has it for itself."""
    c = Case(oracle, fmt, 8, 2, 64, [192, 192, 192], [40, 1, 70], seed=33)
    c.table[1, :2], c.table[2, :2] = c.table[0, :2], c.table[0, :2]
    c.table[2, 2] = c.table[0, 0]  # and one page twice in a sequence
    got = ops.host(c.run(ops))
    check(D.bf16_bits_to_f32(got.view(np.uint16)), *c.want())
    for name in ("k", "v", "ks", "vs"):  # page 1 of sequence 0 is copied for sequence 1
        a = getattr(c.c, name)
        spare = [p for p in range(c.c.pages) if p not in c.table]
        a[spare[0]] = a[c.table[0, 1]]
    c.table[1, 1] = spare[0]
    assert np.array_equal(ops.host(c.run(ops)), got)


@pytest.mark.parametrize("fmt", [None, "fp8"])
def test_captured_and_replayed(oracle, ops, fmt):
    """Graphs with workspaces of their own, on another stream, replayed with other
    inputs and with eager work between."""
    import torch
    cases = [Case(oracle, fmt, 4, 1, 64, [2000, 5] if fmt else [0, 0], [40, 1200], seed=s) for s in (22, 23, 24)]
    dev = [[ops.dev(x) for x in (c.q, c.k, c.v)] for c in cases]
    caches = [c.c.device(ops) if fmt else None for c in cases]
    offs, lengths = ops.dev(cases[0].offs), ops.dev(cases[0].lengths)
    # one table for all, the caches' contents differ
    table = ops.dev(cases[0].table) if fmt else None
    eager = []
    for x, cache in zip(dev, caches):
        ws = ops.prefill_workspace(2, 1240, 4, 1, 64)
        run = (lambda o=None, x=x, cache=cache, ws=ws: ops.kv_prefill(cache, x[0], offs, lengths, table, x[1], x[2], workspace=ws, out=o)
               if cache else ops.attn_prompt(x[0], x[1], x[2], offs, 64, workspace=ws, out=o))
        eager.append((run, ops.host(run())))
    graphs = []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for run, _ in eager[:2]:
        out = torch.zeros((1240, 4, 64), dtype=torch.int16, device="cuda")
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            run(out)
        graphs.append((g, out))
    for _ in range(3):
        for i, (g, out) in enumerate(graphs):
            out.zero_()
            g.replay()
            assert np.array_equal(ops.host(eager[2][0]()), eager[2][1])
            torch.cuda.synchronize()
            assert np.array_equal(ops.host(out), eager[i][1])
    # new inputs in the captured buffers
    for a, b in zip(dev[0], dev[2]):
        a.copy_(b)
    if fmt:
        for name in ("k", "v", "k_scales", "v_scales"):
            getattr(caches[0], name).copy_(getattr(caches[2], name))
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert np.array_equal(ops.host(graphs[0][1]), eager[2][1])


def test_two_streams_at_once(oracle, ops):
    import torch
    cases = [Case(oracle, "int8", 4, 2, 64, [3000, 100], [50, 300], seed=s) for s in (25, 26)]
    want = [ops.host(c.run(ops)) for c in cases]
    state = [([ops.dev(x) for x in (c.q, c.offs, c.lengths, c.table, c.k, c.v)], c.c.device(ops),
              ops.prefill_workspace(2, 350, 4, 2, 64)) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for (x, cache, ws), s in zip(state, streams):
            with torch.cuda.stream(s):
                got.append(ops.kv_prefill(cache, *x, workspace=ws))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert np.array_equal(ops.host(a), b)


def test_empty_calls(ops):
    import torch
    q = torch.zeros((0, 4 * 64), dtype=torch.int16, device="cuda")
    k = torch.zeros((0, 2 * 64), dtype=torch.int16, device="cuda")
    offs = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert ops.attn_prompt(q, k, k, offs, 64).shape == (0, 4, 64)
    q = torch.ones((3, 4 * 64), dtype=torch.int16, device="cuda")
    k = torch.ones((3, 2 * 64), dtype=torch.int16, device="cuda")
    assert not ops.attn_prompt(q, k, k, offs, 64).any()  # rows of no sequence
    offs = torch.zeros(3, dtype=torch.int32, device="cuda")
    assert not ops.attn_prompt(q, k, k, offs, 64).any()


@pytest.mark.parametrize("fmt", [None, "int8"])
@pytest.mark.parametrize("gain", [1.0, 1e4])
@pytest.mark.parametrize("value", ODD)
@pytest.mark.parametrize("token", [5, 700])
def test_odd_values_far_back_reach_who_sees_them(oracle, ops, fmt, gain, value, token):
    """In a tile that whole blocks see, in an early part of split ones: whatever the
    value weighs (with large queries: nothing), split or not."""
    c = Case(oracle, fmt, 2, 2, 64, [1500 if fmt else 0], [2600], seed=34, gain=gain)
    for workspace in (True, False):
        clean = ops.host(c.run(ops, workspace=workspace))
        was = c.v[token, 1, 9]
        c.v[token, 1, 9] = value
        got = ops.host(c.run(ops, workspace=workspace))
        c.v[token, 1, 9] = was
        other = np.ones(got.shape, bool)
        other[token:, 1, 9] = False
        assert np.array_equal(got[other], clean[other])
        hit = D.bf16_bits_to_f32(got.view(np.uint16))[token:, 1, 9]
        assert np.isnan(hit).all() if value == 0x7fc0 else (hit == (np.inf if value == 0x7f80 else -np.inf)).all()


@pytest.mark.parametrize("dim,wide", [(64, False), (61, True), (128, True), (256, False)])
def test_odd_values_of_both_signs(oracle, ops, dim, wide):
    """Infinity from one token on, NaN from the one on that has the other sign; a value of
    another channel, another head and another sequence changes its own alone."""
    c = Case(oracle, None, 2, 1, dim, [0, 0], [40, 900], seed=35, gain=1e3)
    clean = ops.host(c.run(ops))
    c.v[40 + 3, 0, 20], c.v[40 + 500, 0, 20], c.v[40 + 260, 0, dim - 1], c.v[7, 0, 2] = 0x7f80, 0xff80, 0x7fc0, 0xff80
    got = ops.host(c.run(ops, wide=wide, shift=1 if dim % 8 else 8))
    hit = D.bf16_bits_to_f32(got.view(np.uint16))
    assert (hit[43:540, :, 20] == np.inf).all() and np.isnan(hit[540:, :, 20]).all()
    assert np.isnan(hit[300:, :, dim - 1]).all() and (hit[7:40, :, 2] == -np.inf).all()
    other = np.ones(got.shape, bool)
    other[43:, :, 20], other[300:, :, dim - 1], other[7:40, :, 2] = False, False, False
    assert np.array_equal(got[other], clean[other])


@pytest.mark.parametrize("fmt,Hq,H,lengths,new,least", [("fp8", 4, 2, [4000, 64], [20, 300], 1), (None, 2, 1, [0], [2600], 22)])
@pytest.mark.parametrize("slots", [0, 1, 2, 3, 7, 20, 30])
@pytest.mark.parametrize("parts", [-1, 0, 1])
def test_a_workspace_of_some_parts_is_kept_to(oracle, ops, fmt, Hq, H, lengths, new, least, slots, parts):
    """Room for some slots, a part more or less: fewer splits, nothing behind the room.
    least: the slots from which something is split (41 blocks of up to 41 tiles, two parts a slot:
    41 * 41 / 2 slots tiles a part, rounded up past the next whole number, are under 41 from 22 on)."""
    import torch
    c = Case(oracle, fmt, Hq, H, 64, lengths, new, seed=36)
    part = (256 if fmt else 128) * (64 + 2) * 4  # bytes: a workgroup's rows, of padded channels, a maximum and a sum
    room = max((slots * 4 * H + parts) * part, 0)
    usable = room // part // (4 * H)             # whole slots
    buf = torch.full((room + (1 << 20),), 0xa5, dtype=torch.uint8, device="cuda")
    q, k, v = c.args(ops)
    if fmt:
        got = ops.kv_prefill(c.c.device(ops), q, ops.dev(c.offs), ops.dev(c.lengths), ops.dev(c.table), k, v,
                             scale=c.scale, workspace=buf[:room])
    else:
        got = ops.attn_prompt(q, k, v, ops.dev(c.offs), 64, scale=c.scale, workspace=buf[:room])
    check(f32(ops, got), *c.want())
    assert bool((buf[usable * 4 * H * part:] == 0xa5).all())
    assert bool((buf != 0xa5).any()) == (usable >= least)


@pytest.mark.parametrize("fmt,lengths,new", [(None, [0, 0], [300, 70]), ("int8", [3000, 10], [40, 130])])
def test_results_in_the_queries_place(oracle, ops, fmt, lengths, new):
    c = Case(oracle, fmt, 4, 2, 64, lengths, new, seed=37)
    want = ops.host(c.run(ops))
    q, k, v = c.args(ops)
    ws = ops.prefill_workspace(2, len(c.q), 4, 2, 64)
    if fmt:
        ops.kv_prefill(c.c.device(ops), q, ops.dev(c.offs), ops.dev(c.lengths), ops.dev(c.table), k, v, scale=c.scale,
                       workspace=ws, out=q)
    else:
        ops.attn_prompt(q, k, v, ops.dev(c.offs), 64, scale=c.scale, workspace=ws, out=q)
    assert np.array_equal(ops.host(q).reshape(want.shape), want)


def test_results_beside_their_rows_of_one_buffer(oracle, ops):
    """Out in front of and behind the projection's rows, with nothing between."""
    import torch
    c = Case(oracle, None, 4, 2, 64, [0], [90], seed=38)
    want = ops.host(c.run(ops))
    n, size = len(c.q), len(c.q) * 256
    buf = torch.zeros(2 * size + n * 512, dtype=torch.int16, device="cuda")
    rows = buf[size:-size].view(n, 512)
    rows.copy_(ops.dev(np.concatenate([x.reshape(n, -1) for x in (c.q, c.k, c.v)], axis=1)))
    q, k, v = rows.split([256, 128, 128], dim=1)
    for out in (buf[:size], buf[-size:]):
        ops.attn_prompt(q, k, v, ops.dev(c.offs), 64, scale=c.scale, out=out)
        assert np.array_equal(ops.host(out).reshape(want.shape), want)


@pytest.mark.parametrize("width", [0, 3])
def test_a_chunk_of_no_sequences(ops, width):
    """Rows there are, sequences none: zeros, or what out held."""
    import torch
    i16, i32 = dict(dtype=torch.int16, device="cuda"), dict(dtype=torch.int32, device="cuda")
    cache = ops.kv_cache("int8", 4, 2, 64)
    q, k = torch.ones((3, 4 * 64), **i16), torch.ones((3, 2 * 64), **i16)
    args = torch.zeros(1, **i32), torch.zeros(0, **i32), torch.zeros((0, width), **i32)
    assert not ops.kv_prefill(cache, q, *args, k, k).any()
    assert not ops.kv_prefill(cache, q, *args, None, None).any()
    out = torch.full((3, 4, 64), 77, **i16)
    ops.kv_prefill(cache, q, *args, k, k, out=out)
    assert (out == 77).all()


def test_chunks_over_a_table_of_no_pages(oracle, ops):
    """Only the new tokens are seen."""
    c = Case(oracle, "int8", 4, 2, 64, [0, 0], [70, 3], seed=39, width=0)
    assert c.table.shape == (2, 0)
    check(f32(ops, c.run(ops)), *c.want())


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("by", [-100, -110, 110])
def test_value_scales_far_down_and_up(oracle, ops, fmt, by):
    """Weights times scales still are normal bf16 numbers, sums fp32 ones."""
    c = Case(oracle, fmt, 4, 2, 64, [300], [20], seed=43)
    c.c.vs *= np.float32(2.0) ** by
    c.v[:] = 0
    check(f32(ops, c.run(ops)), *c.want())


def test_scores_of_minus_infinity_alone_give_zeros(oracle, ops):
    c = Case(oracle, None, 2, 1, 64, [0], [140], seed=44)
    c.q[..., 0], c.k[:5, 0, 0] = 0x3f80, 0xff80  # the first rows see no other keys
    got = f32(ops, c.run(ops))
    assert not got[:5].any() and np.isfinite(got).all()
