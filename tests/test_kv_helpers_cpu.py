"""The cache's Python helpers: arguments that they must refuse before anything
is enqueued.  No GPU: whatever passes the checks would fail on the launch."""
import pytest
import torch

from longhornai_amd import capi, ops
from tests import _kv
from tests.test_kv_cpu import attn_args

I32 = dict(dtype=torch.int32)


def host_cache():
    c = _kv.HostCache("int8", 4, 2, 40)
    return ops.KvCache("int8", 4, 2, 40, *(torch.from_numpy(a) for a in (c.k, c.v, c.ks, c.vs)))


def call(**kw):
    """kv_attn on six rows of two sequences."""
    a = dict(cache=host_cache(), q=torch.zeros((6, 160), dtype=torch.int16), offsets=torch.tensor([0, 3, 6], **I32),
             lengths=torch.zeros(2, **I32), block_table=torch.zeros((2, 2), **I32),
             k_new=torch.zeros((6, 80), dtype=torch.int16), v_new=torch.zeros((6, 80), dtype=torch.int16))
    a.update(kw)
    return ops.kv_attn(**a)


def test_attn_refuses_a_result_with_rows_that_it_would_leave_unwritten():
    """Six rows of two sequences of at most two tokens: two rows or more would
    hold whatever the new memory held."""
    with pytest.raises(ValueError, match="max_new"):
        call(max_new=2)
    with pytest.raises(ValueError, match="max_new"):
        call(max_new=1, tree=torch.zeros(6, dtype=torch.int64))


@pytest.mark.parametrize("workspace", [torch.zeros(4096, dtype=torch.uint8)[::2],
                                       torch.zeros((64, 64), dtype=torch.float32).t()[:, :32]])
def test_attn_refuses_a_workspace_with_gaps(workspace):
    """The kernels would write the elements between those of the slice."""
    with pytest.raises(ValueError, match="workspace"):
        call(max_new=3, workspace=workspace)


@pytest.mark.parametrize("kw", [dict(offsets=torch.zeros((3, 2), **I32)), dict(lengths=torch.zeros((2, 2), **I32)),
                                dict(lengths=torch.zeros((), **I32)), dict(offsets=torch.zeros((), **I32)),
                                dict(q=torch.zeros(160, dtype=torch.int16)), dict(q=torch.zeros((), dtype=torch.int16)),
                                dict(q=torch.zeros((6, 4, 40, 1), dtype=torch.int16))])
def test_tensors_of_other_ranks(kw):
    """Tables of more than a number a sequence would be read as if they had one."""
    with pytest.raises(ValueError):
        call(max_new=3, **kw)
    if "q" in kw:
        return
    c, k = host_cache(), torch.zeros((6, 80), dtype=torch.int16)
    tables = (kw.get("offsets", torch.tensor([0, 3, 6], **I32)), kw.get("lengths", torch.zeros(2, **I32)),
              torch.zeros((2, 2), **I32))
    with pytest.raises(ValueError):
        ops.kv_write(c, k, k, *tables)
    with pytest.raises(ValueError):
        ops.kv_read(c, *tables, 6)


def test_host_memory_is_refused():
    """Tensors of the host: the kernels would fault on their addresses."""
    c, k = host_cache(), torch.zeros((6, 80), dtype=torch.int16)
    tables = torch.tensor([0, 3, 6], **I32), torch.zeros(2, **I32), torch.zeros((2, 2), **I32)
    with pytest.raises(ValueError, match="GPU"):
        call(max_new=3)
    with pytest.raises(ValueError, match="GPU"):
        ops.kv_write(c, k, k, *tables)
    with pytest.raises(ValueError, match="GPU"):
        ops.kv_read(c, *tables, 6)


@pytest.mark.parametrize("scale", [2.4e38, 3.4e38])
def test_attn_refuses_a_scale_that_is_infinite_as_a_power_of_two(scale):
    """The kernel's weights are powers of two: scale times log2 e must be finite too."""
    args = attn_args(scale=scale)
    assert capi.load().status("lhq_kv_attn_bf16", *args) == capi.LHQ_ERR_INVALID
    assert "scale" in capi.load().last_error()
