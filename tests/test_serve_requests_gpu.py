"""Tables, rotation, attention of chunks and the cache together, as a server runs
them: against 64 bits step by step, and the example."""
import importlib.util
import os

import numpy as np
import pytest

from tests import _data as D
from tests.test_kv_plan_gpu import plan as plan_of
from tests.test_rope_gpu import turned

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example(lib):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "serve_requests.py")
    spec = importlib.util.spec_from_file_location("serve_requests", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("chunk", [256, 65, 1])
def test_the_example(example, fmt, chunk):
    """A weight's and the result's rounding to bf16: each half a step, 2^-8, of what is at most
    the largest value (with chunks of one token kv_attn's, 2^-11)."""
    assert example.main(fmt, chunk) <= 2.0 ** -7


def test_one_step_after_the_other(example):
    """Every step's tables, rotated rows and attention; what is written is read by the next."""
    import torch

    from longhornai_amd import ops
    server = example.Server("int8", 3, 40, seed=5)
    freq = ops.rope_frequencies(example.DIM, theta=500000.0, scaling="yarn", factor=4.0, original=512)
    weight = D.bf16_bits_to_f32(ops.host(server.norms[0], np.uint16))
    g = torch.Generator(device="cuda").manual_seed(3)
    for new in ([200, 1, 0], [64, 1, 130], [1, -1, 1], [1, 300, 1], [-1, 1, 1], [90, 1, 1]):
        n = sum(t for t in new if t > 0)
        x = torch.randn((n, example.HIDDEN), generator=g, device="cuda").to(torch.bfloat16).view(torch.int16)
        table, free, left = (ops.host(t) for t in (server.table, server.free, server.left))
        want = plan_of(server.lengths, new, free, int(left[0]), table, n)
        raw = ops.gemm_w4a16_bf16(x, server.qkv)
        _, o, q, k, v, plan = server.step(x, new)
        for a, b in zip((plan.offsets, plan.positions, plan.slots, plan.left, server.table, server.free), want):
            assert np.array_equal(ops.host(a), b)
        raw = D.bf16_bits_to_f32(ops.host(raw, np.uint16))
        H, W = example.HEADS, example.KV_HEADS
        for got, lo, heads in ((q, 0, H), (k, H, W)):
            y, bound = turned(raw[:, lo * 128:(lo + heads) * 128].reshape(n, heads, 128), want[1], freq, False,
                              server.turns.gain, weight, 1e-6, 8)
            y2 = D.bf16_bits_to_f32(ops.host(got.contiguous(), np.uint16)).reshape(y.shape)
            assert (np.abs(y2 - y) <= bound).all()
        at = 0
        for s, t in enumerate(new):
            if t > 0:
                rows = slice(at, at + t)
                exact = server.attended(s, int(server.lengths[s]), q[rows], k[rows], v[rows])
                got = o[rows].view(torch.bfloat16).double().cpu().numpy()
                assert np.abs(got - exact).max() <= 2.0 ** -7 * np.abs(exact).max()
                server.lengths[s] += t
                at += t
            elif t < 0:
                server.lengths[s] = 0
