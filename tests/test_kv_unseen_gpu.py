"""Attention over the 8-bit cache: values of new tokens that a query does not
see, of any size, change nothing of its result; seen ones of any size and weight
keep the others' precision.  Against 64-bit numpy (tests/_kv.py) and bit for bit
against the same call with ordinary values in the unseen places."""
import numpy as np
import pytest

from tests import _data as D
from tests import _kv
from tests.test_kv_gpu import Case, rng

pytestmark = pytest.mark.gpu

# 2^40, 2^60, the largest of either sign, a subnormal: finite bf16 patterns that unwritten memory may hold
SIZES = (0x5380, 0x5d80, 0x7f7f, 0xff7f, 0x0001)


@pytest.fixture(scope="module")
def ops(lib):
    from longhornai_amd import ops as _ops
    return _ops


def words(T, of):
    """Row masks of a tree of T tokens: bit j of row i where of(i, j)."""
    return np.array([sum(1 << j for j in range(T) if of(i, j)) for i in range(T)], np.uint64)


def same_but(c, T, hidden, seen_by):
    """Runs c with ordinary values, then with each size in the `hidden` tokens of
    every sequence: rows that see none of them must not change by a bit, all
    rows hold to 64 bits."""
    n = len(c.new)
    at = (np.arange(n)[:, None] * T + np.asarray(hidden)).reshape(-1)
    blind = [s * T + i for s in range(n) for i in range(T) if not seen_by(i)]
    clean = c.ops.host(c.run(), np.uint16).copy()
    c.check()
    ordinary = c.v.copy()
    for bits in SIZES:
        c.v[at] = bits
        got = c.ops.host(c.run(), np.uint16)
        assert np.array_equal(got[blind], clean[blind]), hex(bits)
        c.check()
        c.v[...] = ordinary


@pytest.mark.parametrize("T", [2, 3, 33, 64])
@pytest.mark.parametrize("fmt,Hq,H,Dh", [("int8", 8, 2, 128), ("fp8", 3, 1, 64), ("int8", 2, 1, 256)])
def test_padding_rows(oracle, ops, fmt, Hq, H, Dh, T):
    """The last third of a tree is padding that no row sees, itself included;
    cached tokens on the same waves, and none."""
    real = T - max(1, T // 3)
    c = Case(oracle, ops, fmt, Hq, H, Dh, [700, 0, 1100], [T] * 3, seed=T)
    c.tree = np.tile(words(T, lambda i, j: j <= i and j < real), 3)
    same_but(c, T, range(real, T), lambda i: False)


@pytest.mark.parametrize("T", [2, 3, 33, 64])
@pytest.mark.parametrize("fmt,Hq,H,Dh", [("fp8", 8, 2, 128), ("int8", 16, 1, 96), ("fp8", 2, 1, 256)])
def test_masked_siblings(oracle, ops, fmt, Hq, H, Dh, T):
    """Every second token is a leaf that only its own row sees, beside the root
    and the cached tokens."""
    c = Case(oracle, ops, fmt, Hq, H, Dh, [700, 0, 1100], [T] * 3, seed=T + 1)
    c.tree = np.tile(words(T, lambda i, j: j == i or (j % 2 == 0 and j < i)), 3)
    same_but(c, T, range(1, T, 2), lambda i: i % 2 == 1)


@pytest.mark.parametrize("new", [1, 2, 40])
def test_rows_that_see_only_the_cache(oracle, ops, new):
    """Empty masks beside rows that see everything."""
    c = Case(oracle, ops, "int8", 4, 2, 64, [300, 64, 1], [new + 1] * 3, seed=new)
    c.tree = np.tile(words(new + 1, lambda i, j: i > 0), 3)
    same_but(c, new + 1, range(new + 1), lambda i: i > 0)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("T", [4, 40])
def test_seen_values_of_little_weight(oracle, ops, fmt, T):
    """A token that every row sees, with values of 2^60 and a score so low that
    its share of a result is under 2^-60: the others keep their precision.  No
    cached tokens, whose scales share an exponent."""
    c = Case(oracle, ops, fmt, 4, 1, 64, [0, 0], [T, T], seed=T, tree=False)
    first = c.offs[:-1]
    c.q[..., 0], c.k[first, :, 0] = 0x4140, 0xc440  # 12, -768: a score of -1152, e^-1152 under 2^-1660
    c.v[first] = 0x5d80
    c.q[first], c.k[first, :, 0] = 0, 0xc440        # (the first row sees itself alone: its score is zero)
    want, bound = c.want()
    got = D.bf16_bits_to_f32(ops.host(c.run(), np.uint16))
    # the oracle's bound without its term of the largest value, whatever its weight: 2^-30 of the largest other one
    rest = np.ones(len(c.q), bool)
    rest[first] = False
    big = np.abs(D.bf16_bits_to_f32(c.v)[rest]).max()
    tight = np.where(rest[:, None, None], np.minimum(bound, 2.0 ** -7 * np.abs(want) + 2.0 ** -10 * big), bound)
    assert (np.abs(got - want) <= tight).all()


def test_new_values_from_subnormal_to_largest(oracle, ops):
    """Value rows whose sizes step from 2^-110 to 2^126 down a chain, and up it;
    with and without cached tokens."""
    T = 64
    for order in (1, -1):
        for lengths in ([0, 0], [200, 64]):
            c = Case(oracle, ops, "int8", 8, 2, 64, lengths, [T, T], seed=5, tree=False)
            size = np.exp2(np.linspace(-110, 126, T))[::order]
            x = rng(3).uniform(0.5, 1.0, c.v.shape) * np.tile(size, 2)[:, None, None]
            c.v = D.to_bf16_bits(oracle, x.astype(np.float32)).reshape(c.v.shape)
            c.check()
