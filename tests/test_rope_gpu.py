"""Turned and normed heads on the GPU against 64-bit numpy."""
import numpy as np
import pytest

from tests import _data as D

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(lib):
    from longhornai_amd import ops as _ops
    return _ops


def turned(x, positions, freq, interleaved, gain, weight, eps, bits):
    """(y, bound) in 64 bits.  The bound, with (a, b) the pair that y is made of:
      2^-8 |y| or 2^-24 |y|      rounding to bf16, or to fp32
      (|a| + |b|) gain 2^-20     fp32 before it, 16 half steps: an angle of under pi / 4 off by 3
                                 roundings of itself, 2 of the series, cosine times gain 1, the
                                 norm's factor and the weight 3, two products and their sum 3; the
                                 rest of 2^-64 turns and of the position's whole turns is under 1"""
    n, H, dim = x.shape
    x = x.astype(np.float64)
    if weight is not None:
        x = x / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps) * weight.astype(np.float64)
    rot = 2 * len(freq)
    angle = positions.astype(np.float64)[:, None] * freq
    c, s = np.cos(angle)[:, None] * gain, np.sin(angle)[:, None] * gain
    y, size = x.copy(), np.abs(x)
    at = (np.arange(0, rot, 2), np.arange(1, rot, 2)) if interleaved else (np.arange(rot // 2), np.arange(rot // 2, rot))
    a, b = x[..., at[0]], x[..., at[1]]
    y[..., at[0]], y[..., at[1]] = a * c - b * s, b * c + a * s
    size[..., at[0]] = size[..., at[1]] = (np.abs(a) + np.abs(b)) * abs(gain)
    return y, np.abs(y) * 2.0 ** -bits + size * 2.0 ** -20


class Case:
    def __init__(self, oracle, ops, dtype, n, Hq, H, dim, norm, seed, reach=5000, **plan):
        g = np.random.default_rng(seed)
        self.bf16, self.Hq, self.H, self.dim = dtype == "bf16", Hq, H, dim

        def some(shape, by=1.0):
            x = (g.standard_normal(shape) * by).astype(np.float32)
            return D.to_bf16_bits(oracle, x) if self.bf16 else x
        self.q, self.k = some((n, Hq, dim), 2.0), some((n, H, dim))
        self.qw, self.kw = (some(dim, 0.5), some(dim, 0.5)) if norm else (None, None)
        self.pos = g.integers(0, reach, n).astype(np.int32)
        self.plan = ops.rope_plan(dim, **plan)
        kw = {k: v for k, v in plan.items() if k not in ("rot_dim", "interleaved", "gain")}
        self.freq = ops.rope_frequencies(self.plan.rot_dim, **kw)

    def value(self, x):
        return None if x is None else D.bf16_bits_to_f32(x) if self.bf16 else x

    def want(self, eps=1e-6):
        return [turned(self.value(x), self.pos, self.freq, self.plan.interleaved, self.plan.gain, self.value(w), eps,
                       8 if self.bf16 else 24) for x, w in ((self.q, self.qw), (self.k, self.kw))]

    def run(self, ops, eps=1e-6, **kw):
        w = [None if x is None else ops.dev(x) for x in (self.qw, self.kw)]
        q, k = ops.rope(self.plan, ops.dev(self.q), ops.dev(self.k), ops.dev(self.pos), q_weight=w[0], k_weight=w[1],
                        eps=eps, **kw)
        return self.host(ops, q), self.host(ops, k)

    def host(self, ops, t):
        return D.bf16_bits_to_f32(ops.host(t, np.uint16)) if self.bf16 else ops.host(t)

    def check(self, got, eps=1e-6):
        for y, (want, bound) in zip(got, self.want(eps)):
            assert (np.abs(y - want) <= bound).all(), float((np.abs(y - want) - bound).max())


SHAPES = [(1, 1, 1, 2, {}), (3, 2, 1, 1, {}), (5, 3, 1, 7, dict(rot_dim=4)), (70, 4, 2, 64, {}), (33, 15, 5, 80, dict(rot_dim=40)),
          (9, 8, 2, 128, {}), (17, 8, 2, 128, dict(rot_dim=64)), (6, 4, 1, 96, dict(rot_dim=30)), (4, 2, 2, 256, {}),
          (5, 6, 2, 192, dict(rot_dim=128)), (8, 5, 1, 255, dict(rot_dim=254)), (3, 4, 4, 40, dict(rot_dim=0)),
          (300, 32, 8, 128, {}), (2, 40, 40, 72, dict(rot_dim=48))]


@pytest.mark.parametrize("n,Hq,H,dim,kw", SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_shapes(oracle, ops, dtype, n, Hq, H, dim, kw, interleaved, norm):
    kw = dict(rot_dim=dim - dim % 2, **kw) if "rot_dim" not in kw else kw
    c = Case(oracle, ops, dtype, n, Hq, H, dim, norm, seed=dim, interleaved=interleaved, **kw)
    c.check(c.run(ops))


@pytest.mark.parametrize("scaling", [None, "linear", "ntk", "yarn"])
def test_scaled_frequencies_at_far_positions(oracle, ops, scaling):
    """Positions up to a million, whose angle fp32 has not to a radian's tenth."""
    c = Case(oracle, ops, "f32", 200, 4, 2, 128, True, seed=1, reach=1 << 20, theta=500000.0, scaling=scaling, factor=8.0)
    c.check(c.run(ops))


def test_whole_turns_fall_away(oracle, ops):
    """A pair of a quarter turn per position is exact at any of them, 2^31 - 1 too."""
    import torch
    plan = ops.RopePlan(2, 2, torch.tensor([1 << 62], device="cuda"), False, 1.0)
    pos = np.array([0, 1, 2, 3, 2 ** 31 - 1, 2 ** 31 - 2, 2 ** 30], np.int32)
    x = np.tile(np.float32([3.0, 5.0]), (7, 1, 1))
    got, _ = ops.rope(plan, ops.dev(x), None, ops.dev(pos))
    turns = {0: (3, 5), 1: (-5, 3), 2: (-3, -5), 3: (5, -3)}
    assert np.allclose(ops.host(got)[:, 0], [turns[p % 4] for p in pos.tolist()], atol=8 * 2.0 ** -22, rtol=0)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dim,shift", [(64, 0), (64, 3), (128, 8), (80, 4)])
def test_in_place_in_slices_of_one_projection(oracle, ops, dtype, dim, shift):
    import torch
    c = Case(oracle, ops, dtype, 50, 6, 2, dim, True, seed=2)
    want = c.run(ops)
    width = 10 * dim + shift
    buf = ops.dev(np.full(50 * width + shift, 9, c.q.dtype.type if c.bf16 else np.float32))
    rows = buf[shift:].view(50, width)
    q, k, v = rows[:, :10 * dim].split([6 * dim, 2 * dim, 2 * dim], dim=1)
    q.copy_(ops.dev(c.q).view(50, -1))
    k.copy_(ops.dev(c.k).view(50, -1))
    got = ops.rope(c.plan, q, k, ops.dev(c.pos), q_weight=ops.dev(c.qw), k_weight=ops.dev(c.kw), out=(q, k))
    assert got[0] is q and got[1] is k
    assert np.array_equal(c.host(ops, q.contiguous()).reshape(want[0].shape), want[0])
    assert np.array_equal(c.host(ops, k.contiguous()).reshape(want[1].shape), want[1])
    assert torch.equal(v, torch.full_like(v, 9)) and bool((rows[:, 10 * dim:] == 9).all())


def test_rows_without_a_position_are_passed_on(oracle, ops):
    c = Case(oracle, ops, "bf16", 40, 4, 2, 128, True, seed=3)
    c.pos[[0, 17, 39]] = [-1, -2 ** 31, -5]
    q, k = c.run(ops)
    c.pos = np.maximum(c.pos, 0)
    for y, x, (want, bound) in zip((q, k), (c.q, c.k), c.want()):
        some = np.ones(40, bool)
        some[[0, 17, 39]] = False
        assert np.array_equal(y[~some], D.bf16_bits_to_f32(x[~some]))
        assert (np.abs(y - want) <= bound)[some].all()


# channels that are cut into vectors of 8, 4, 2 and 1, and into none; more heads than a lane has at a time
CUTS = [(2, 2), (6, 4), (40, 40), (40, 20), (64, 62), (100, 100), (100, 50), (128, 126), (126, 126), (130, 130),
        (144, 136), (192, 188), (250, 250), (254, 126), (256, 252), (256, 254), (33, 32)]


@pytest.mark.parametrize("dim,rot", CUTS)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_channels_of_any_number(oracle, ops, dtype, dim, rot, interleaved, norm):
    c = Case(oracle, ops, dtype, 19, 41, 27, dim, norm, seed=dim, rot_dim=rot, interleaved=interleaved)
    c.check(c.run(ops))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dim,rot", [(40, 40), (128, 126), (100, 100)])
def test_any_number_in_place_in_odd_slices(oracle, ops, dtype, dim, rot):
    c = Case(oracle, ops, dtype, 50, 6, 2, dim, True, seed=6, rot_dim=rot)
    want = c.run(ops)
    width = 8 * dim + 3
    buf = ops.dev(np.full(50 * width + 1, 9, c.q.dtype.type if c.bf16 else np.float32))
    rows = buf[1:].view(50, width)
    q, k, rest = rows.split([6 * dim, 2 * dim, 3], dim=1)
    q.copy_(ops.dev(c.q).view(50, -1))
    k.copy_(ops.dev(c.k).view(50, -1))
    w = (None if x is None else ops.dev(x) for x in (c.qw, c.kw))
    got = ops.rope(c.plan, q, k, ops.dev(c.pos), *w, out=(q, k))
    for g, x in zip(got, want):
        assert np.array_equal(c.host(ops, g.contiguous()).reshape(x.shape), x)
    assert (ops.host(rest.contiguous()) == 9).all() and ops.host(buf)[0] == 9


@pytest.mark.parametrize("side", ["q", "k"])
def test_one_side_alone(oracle, ops, side):
    c = Case(oracle, ops, "bf16", 30, 4, 2, 64, False, seed=4)
    both = c.run(ops)
    q, k = (ops.dev(c.q), None) if side == "q" else (None, ops.dev(c.k))
    got = ops.rope(c.plan, q, k, ops.dev(c.pos))
    i = 0 if side == "q" else 1
    assert got[1 - i] is None and np.array_equal(c.host(ops, got[i]), both[i])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("by", [1e-30, 1e-18, 1e18, 1e30])
def test_norms_of_every_size(oracle, ops, dtype, by):
    """Sums of squares outside fp32's range; eps is far below them or far above."""
    c = Case(oracle, ops, dtype, 20, 4, 2, 64, True, seed=5)
    c.q, c.k = ((D.to_bf16_bits(oracle, (c.value(x) * np.float32(by)).astype(np.float32)) if c.bf16 else
                 (x * np.float32(by)).astype(np.float32)) for x in (c.q, c.k))
    for eps in (0.0, 1e-6):
        c.check(c.run(ops, eps=eps), eps=eps)


def test_heads_of_zeros(oracle, ops):
    c = Case(oracle, ops, "bf16", 3, 2, 1, 64, True, seed=6)
    c.q[:], c.k[1] = 0, 0
    q, k = c.run(ops)
    assert not q.any() and not k[1].any() and k[0].any()


def test_values_that_are_not_finite_stay_in_their_pair(oracle, ops):
    c = Case(oracle, ops, "f32", 4, 2, 1, 64, False, seed=7)
    clean, _ = c.run(ops)
    c.q[1, 1, 5] = np.nan
    got, _ = c.run(ops)
    hit = np.zeros(got.shape, bool)
    hit[1, 1, [5, 37]] = True
    assert np.isnan(got[hit]).all() and np.array_equal(got[~hit], clean[~hit])


def test_captured_and_replayed(oracle, ops):
    import torch
    c = Case(oracle, ops, "bf16", 64, 8, 2, 128, True, seed=8)
    want = c.run(ops)
    q, k, pos, qw, kw = (ops.dev(x) for x in (c.q, c.k, c.pos, c.qw, c.kw))
    out = (torch.zeros_like(q), torch.zeros_like(k))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.rope(c.plan, q, k, pos, q_weight=qw, k_weight=kw, out=out)
    for _ in range(3):
        out[0].zero_()
        g.replay()
        assert np.array_equal(c.run(ops)[0], want[0])
        torch.cuda.synchronize()
        assert np.array_equal(c.host(ops, out[0]), want[0]) and np.array_equal(c.host(ops, out[1]), want[1])


def test_no_rows(ops):
    import torch
    plan = ops.rope_plan(64)
    q, k = (torch.zeros((0, h * 64), dtype=torch.int16, device="cuda") for h in (4, 2))
    got = ops.rope(plan, q, k, torch.zeros(0, dtype=torch.int32, device="cuda"), out=(q, k))
    assert got[0].shape == (0, 256)


@pytest.mark.parametrize("interleaved", [False, True])
def test_frequencies_of_the_callers(oracle, ops, interleaved):
    """Any of them: faster than a turn a position, backwards, none."""
    c = Case(oracle, ops, "f32", 50, 3, 1, 64, False, seed=40, reach=3000, interleaved=interleaved)
    f = np.random.default_rng(41).normal(0.0, 4.0, 32)
    f[5] = 0.0
    c.freq, c.plan = f, ops.rope_plan(64, interleaved=interleaved, frequencies=f)
    c.check(c.run(ops))


@pytest.mark.parametrize("n", [1, 2])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_in_place_by_views_of_heads(oracle, ops, dtype, n):
    """Slices of one projection as [n, heads, dim]: of one row such a view has a stride of its own."""
    import torch
    c = Case(oracle, ops, dtype, n, 4, 2, 64, True, seed=42)
    want = c.run(ops)
    wide = torch.cat([ops.dev(x).reshape(n, -1) for x in (c.q, c.k)], dim=1)
    q, k = wide.split([256, 128], dim=1)
    out = q.view(n, 4, 64), k.view(n, 2, 64)
    w = [ops.dev(x) for x in (c.qw, c.kw)]
    ops.rope(c.plan, q, k, ops.dev(c.pos), q_weight=w[0], k_weight=w[1], out=out)
    for got, x in zip(out, want):
        assert np.array_equal(c.host(ops, got.contiguous()), x)
