"""The cache's Python helpers on the GPU: what their defaults compute."""
import numpy as np
import pytest

from tests import _data as D
from tests.test_kv_gpu import Case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(lib):
    from longhornai_amd import ops as _ops
    return _ops


def attn(ops, c, **kw):
    return ops.kv_attn(c.c.device(ops), ops.dev(c.q), ops.dev(c.offs), ops.dev(c.lengths), ops.dev(c.table),
                       ops.dev(c.k), ops.dev(c.v), scale=c.scale,
                       tree=None if c.tree is None else ops.dev(c.tree.view(np.int64)), **kw)


@pytest.mark.parametrize("new", [[1, 1, 1], [5, 0, 12], [64], [40, 64, 3]])
def test_without_max_new_every_row_is_computed(oracle, ops, new):
    c = Case(oracle, ops, "int8", 4, 2, 64, [100, 30, 0][:len(new)], new, seed=3)
    want, bound = c.want()
    got = D.bf16_bits_to_f32(ops.host(attn(ops, c), np.uint16))
    assert (np.abs(got - want) <= bound).all()


def test_without_max_new_rows_past_the_64th_of_a_sequence_are_zeros(oracle, ops):
    """More than 64 new tokens of one sequence: those that no call computes."""
    import torch
    c = Case(oracle, ops, "int8", 4, 2, 64, [100, 30], [70, 5], seed=3, tree=False)
    for _ in range(3):  # (memory that the allocator hands out again holds this)
        torch.full(c.q.shape, 77, dtype=torch.int16, device="cuda")
    got = ops.host(attn(ops, c), np.uint16)
    c.new = [70, 5]
    ref = ops.host(c.run(max_new=64, out=ops.zeros(c.q.shape, np.int16)), np.uint16)
    assert not got[64:70].any() and np.array_equal(got, ref) and got[:64].any() and got[70:].any()


def test_without_max_new_rows_of_no_sequence_are_zeros(oracle, ops):
    """Offsets that begin after the first row and end before the last."""
    import torch
    c = Case(oracle, ops, "int8", 4, 2, 64, [100, 30], [2, 5], seed=3, tree=False)
    for _ in range(3):
        torch.full(c.q.shape, 77, dtype=torch.int16, device="cuda")
    c.offs = np.array([1, 3, 6], np.int32)
    got = ops.host(attn(ops, c), np.uint16)
    want, bound = c.want()
    assert (np.abs(D.bf16_bits_to_f32(got) - want) <= bound).all()
    assert not got[0].any() and not got[6].any() and got[1:6].any(axis=(1, 2)).all()
