"""Tables, rotation and attention of prompts without a GPU: sizes, refusals of the
C ABI and of the Python helpers, frequencies, the tests' oracle."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from longhornai_amd import capi, ops
from tests import _kv, _prefill

FAKE, ODD = C.c_void_p(0x1000), C.c_void_p(0x1004)  # never dereferenced: validation fails first
INV, UNS = capi.LHQ_ERR_INVALID, capi.LHQ_ERR_UNSUPPORTED


@pytest.fixture(scope="module")
def L():
    return capi.load()


def plan_args(**kw):
    a = dict(lengths=FAKE, new=FAKE, tree=None, left=FAKE, left_out=FAKE, free=FAKE, table=FAKE, offsets=FAKE,
             positions=FAKE, slots=FAKE, seqs=3, cap=5, width=4, pages=9, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(seqs=-1), INV), (dict(cap=-1), INV), (dict(width=-1), INV), (dict(pages=-1), INV), (dict(width=1 << 25), UNS),
    (dict(cap=2 ** 31 - 1), UNS), (dict(seqs=2 ** 31 - 1), UNS), (dict(lengths=None), INV), (dict(new=None), INV), (dict(left=None), INV),
    (dict(left_out=None), INV), (dict(free=None), INV), (dict(table=None), INV), (dict(offsets=None), INV),
    (dict(positions=None), INV)])
def test_plan_refusals(L, kw, code):
    assert L.status("lhq_kv_plan", *plan_args(**kw)) == code, L.last_error()
    assert "kv_plan" in L.last_error()


def rope_args(**kw):
    a = dict(q=C.c_void_p(1 << 20), qs=1024, k=C.c_void_p(2 << 20), ks=256, pos=FAKE, turns=FAKE, qw=None, kw=None,
             eps=C.c_float(1e-6), gain=C.c_float(1.0), qo=C.c_void_p(3 << 20), qos=1024, ko=C.c_void_p(4 << 20), kos=256,
             inter=0, n=7, heads=8, kv=2, D=128, rot=128, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("fn", ["lhq_rope_f32", "lhq_rope_bf16"])
@pytest.mark.parametrize("kw,code", [
    (dict(n=-1), INV), (dict(n=(1 << 23) + 1), UNS), (dict(heads=-1), INV), (dict(kv=-1), INV), (dict(D=0), INV),
    (dict(D=257, qs=9999, ks=9999, qos=9999, kos=9999), UNS), (dict(heads=70000), UNS), (dict(rot=127), INV),
    (dict(rot=130), INV), (dict(rot=-2), INV), (dict(inter=2), INV), (dict(eps=C.c_float(-1e-6)), INV),
    (dict(eps=C.c_float(math.nan)), INV), (dict(gain=C.c_float(math.inf)), INV), (dict(qs=1023), INV), (dict(ks=255), INV),
    (dict(qos=1023), INV), (dict(kos=-256), INV), (dict(q=None), INV), (dict(ko=None), INV), (dict(pos=None), INV),
    (dict(turns=None), INV),
    # results over inputs, or over each other, without being in place
    (dict(qo=C.c_void_p((1 << 20) + 8)), INV), (dict(qo=C.c_void_p(1 << 20), qos=1032), INV),
    (dict(qo=C.c_void_p(2 << 20)), INV), (dict(ko=C.c_void_p(1 << 20)), INV), (dict(ko=C.c_void_p((3 << 20) + 64)), INV)])
def test_rope_refusals(L, fn, kw, code):
    assert L.status(fn, *rope_args(**kw)) == code, L.last_error()
    assert fn[4:] in L.last_error()


def test_rope_with_nothing_to_do_is_ok(L):
    assert L.status("lhq_rope_bf16", *rope_args(n=0, q=None, pos=None)) == 0
    assert L.status("lhq_rope_f32", *rope_args(heads=0, kv=0, q=None, k=None)) == 0


def prompt_args(**kw):
    a = dict(q=FAKE, qs=4096, k=FAKE, ks=1024, v=FAKE, vs=1024, offsets=FAKE, out=FAKE, seqs=2, cap=5, heads=32, kv=8,
             D=128, scale=C.c_float(0.1), rest=0, ws=None, wsb=0, stream=None)
    a.update(kw)
    return list(a.values())


def prefill_args(**kw):
    a = dict(q=FAKE, qs=4096, k=FAKE, ks=1024, v=FAKE, vs=1024, offsets=FAKE, lengths=FAKE, table=FAKE, kc=FAKE, ksc=FAKE,
             vc=FAKE, vsc=FAKE, out=FAKE, fmt=0, seqs=2, cap=5, width=4, pages=9, heads=32, kv=8, D=128,
             scale=C.c_float(0.1), rest=0, ws=None, wsb=0, stream=None)
    a.update(kw)
    return list(a.values())


COMMON = [(dict(seqs=-1), INV), (dict(cap=-1), INV), (dict(D=0), INV), (dict(D=257, qs=9999, ks=9999, vs=9999), UNS),
          (dict(kv=0), INV), (dict(heads=30), INV), (dict(heads=0), INV), (dict(heads=-8), INV),
          (dict(heads=80000, qs=1 << 40), UNS), (dict(cap=1 << 27), UNS), (dict(scale=C.c_float(0.0)), INV),
          (dict(scale=C.c_float(-1.0)), INV), (dict(scale=C.c_float(math.nan)), INV), (dict(scale=C.c_float(math.inf)), INV),
          (dict(scale=C.c_float(3e38)), INV), (dict(k=None), INV), (dict(v=None), INV), (dict(qs=4095), INV),
          (dict(ks=1000), INV), (dict(vs=1000), INV), (dict(wsb=-1), INV), (dict(ws=ODD, wsb=1 << 20), INV),
          (dict(q=None), INV), (dict(out=None), INV), (dict(offsets=None), INV)]


@pytest.mark.parametrize("kw,code", COMMON + [(dict(k=None, v=None), INV)])
def test_prompt_refusals(L, kw, code):
    assert L.status("lhq_attn_prompt_bf16", *prompt_args(**kw)) == code, L.last_error()
    assert "attn_prompt" in L.last_error()


@pytest.mark.parametrize("kw,code", COMMON + [
    (dict(fmt=2), INV), (dict(fmt=-1), INV), (dict(width=-1), INV), (dict(pages=-1), INV), (dict(width=1 << 25), UNS),
    (dict(lengths=None), INV), (dict(table=None), INV), (dict(kc=None), INV), (dict(ksc=None), INV), (dict(vc=None), INV),
    (dict(vsc=None), INV), (dict(kc=ODD), INV), (dict(vc=ODD), INV), (dict(ksc=ODD), INV), (dict(vsc=ODD), INV)])
def test_prefill_refusals(L, kw, code):
    assert L.status("lhq_kv_prefill_bf16", *prefill_args(**kw)) == code, L.last_error()
    assert "kv_prefill" in L.last_error()


def test_attention_with_nothing_to_do_is_ok(L):
    for kw in (dict(seqs=0), dict(cap=0)):
        assert L.status("lhq_attn_prompt_bf16", *prompt_args(q=None, **kw)) == 0
        assert L.status("lhq_kv_prefill_bf16", *prefill_args(q=None, **kw)) == 0


def test_workspace_sizes(L):
    ws = L.lhq_prefill_workspace_bytes
    assert ws(1, 100000, 32, 8, 128) == 0         # rows enough for the chip
    assert ws(1, 64, 32, 8, 128) > 0
    assert ws(1, 64, 32, 8, 128) % 16 == 0
    # a part has as many rows as there can be, at most those of a workgroup
    assert ws(1, 1, 8, 8, 128) * 4 == ws(1, 4, 8, 8, 128)
    assert ws(1, 64, 32, 8, 128) == ws(1, 65, 32, 8, 128)
    for bad in ((0, 4, 8, 8, 64), (4, 0, 8, 8, 64), (4, 4, 9, 8, 64), (4, 4, 8, 0, 64), (4, 4, 8, 8, 300), (4, 4, 0, 8, 64),
                (-1, 4, 8, 8, 64), (4, 4, 8, 8, 0)):
        assert ws(*bad) == 0


def test_plan_helper_refusals():
    i32 = dict(dtype=torch.int32)
    good = dict(lengths=torch.zeros(2, **i32), new_tokens=torch.ones(2, **i32), free_pages=torch.zeros(5, **i32),
                left=torch.zeros(2, **i32), block_table=torch.zeros((2, 3), **i32), n=2)
    for kw in (dict(lengths=torch.zeros(3, **i32)), dict(new_tokens=torch.ones(2, dtype=torch.int64)),
               dict(free_pages=torch.zeros((5, 1), **i32)), dict(left=torch.zeros(1, **i32)), dict(block_table=torch.zeros(6, **i32)),
               dict(block_table=torch.zeros((2, 6), **i32)[:, ::2]), dict(n=-1), dict(tree=torch.zeros(3, dtype=torch.int64)),
               dict(free_pages=torch.zeros(10, **i32)[::2]),
               dict(out=ops.KvPlan(*(torch.zeros(k, **i32) for k in (3, 2, 2, 2)))),
               {}):  # (nothing wrong but that it is not on a GPU)
        with pytest.raises(ValueError):
            ops.kv_plan(**{**good, **kw})


def test_rope_helper_refusals():
    plan = ops.RopePlan(64, 64, torch.zeros(32, dtype=torch.int64), False, 1.0)
    q, k = torch.zeros((3, 256), dtype=torch.int16), torch.zeros((3, 128), dtype=torch.int16)
    pos = torch.zeros(3, dtype=torch.int32)
    w = torch.zeros(64, dtype=torch.int16)
    for args, kw in (((None, None, pos), {}), ((q[:, :200], k, pos), {}), ((q, k[:2], pos), {}), ((q, k.float(), pos), {}),
                     ((q.double(), None, pos), {}), ((q, k, pos[:2]), {}), ((q, k, pos.long()), {}),
                     ((q, k, pos), dict(q_weight=w.float())), ((q, k, pos), dict(k_weight=w[:32])),
                     ((q, None, pos), dict(k_weight=w)), ((q, k, pos), dict(out=(q, None))),
                     ((q, k, pos), dict(out=(q[:2], k))), ((q, k, pos), dict(out=(q.float(), k))), ((q, k, pos), {})):
        with pytest.raises(ValueError):
            ops.rope(plan, *args, **kw)


def test_attention_helper_refusals():
    i32 = dict(dtype=torch.int32)
    c = _kv.HostCache("int8", 4, 2, 40)
    cache = ops.KvCache("int8", 4, 2, 40, *(torch.from_numpy(x) for x in (c.k, c.v, c.ks, c.vs)))
    q, k = torch.zeros((6, 160), dtype=torch.int16), torch.zeros((6, 80), dtype=torch.int16)
    offs, start, table = torch.tensor([0, 3, 6], **i32), torch.zeros(2, **i32), torch.zeros((2, 2), **i32)
    for a, kw in (((q, k, k[:5]), {}), ((q, k[:, :79], k), {}), ((q.float(), k, k), {}), ((q[:, :120], k, k), {}),
                  ((q, k, None), {}), ((q, k, k), dict(out=torch.zeros((6, 4, 40)))),
                  ((q, k, k), dict(out=torch.zeros((5, 4, 40), dtype=torch.int16))),
                  ((q, k, k), dict(workspace=torch.zeros((8, 8))[:, ::2])), ((q, k, k), {})):
        with pytest.raises(ValueError):
            ops.attn_prompt(*a, offs, 40, **kw)
        with pytest.raises(ValueError):
            ops.kv_prefill(cache, a[0], offs, start, table, a[1], a[2], **kw)
    for bad in (offs.long(), offs[None], offs[:0], torch.zeros(6, **i32)[::2]):
        with pytest.raises(ValueError):
            ops.attn_prompt(q, k, k, bad, 40)
        with pytest.raises(ValueError):
            ops.kv_prefill(cache, q, bad, start, table, k, k)
    for bad in (start.long(), torch.zeros(3, **i32)):
        with pytest.raises(ValueError):
            ops.kv_prefill(cache, q, offs, bad, table, k, k)
    with pytest.raises(ValueError):  # the cache's kv heads, not the rows'
        ops.kv_prefill(cache, q, offs, start, table, k[:, :40], k[:, :40])


def test_frequencies():
    f = ops.rope_frequencies(8, theta=10000.0)
    assert np.allclose(f, [1, 0.1, 0.01, 0.001], rtol=1e-14)
    assert np.allclose(ops.rope_frequencies(8, scaling="linear", factor=4.0), f / 4, rtol=1e-14)
    ntk = ops.rope_frequencies(8, scaling="ntk", factor=4.0)
    assert ntk[0] == 1 and math.isclose(ntk[-1], f[-1] / 4, rel_tol=1e-12)
    yarn = ops.rope_frequencies(64, scaling="yarn", factor=4.0, original=4096)
    plain = ops.rope_frequencies(64)
    turns = 4096 * plain / (2 * math.pi)
    assert np.allclose(yarn[turns > 32], plain[turns > 32]) and np.allclose(yarn[turns < 1], plain[turns < 1] / 4)
    assert (yarn <= plain * (1 + 1e-12)).all() and (yarn >= plain / 4 * (1 - 1e-12)).all()
    for kw in (dict(rot_dim=7), dict(rot_dim=-2), dict(rot_dim=8, theta=0.5), dict(rot_dim=8, theta=math.nan),
               dict(rot_dim=8, factor=0.0), dict(rot_dim=8, scaling="log"), dict(rot_dim=2, scaling="ntk"),
               dict(rot_dim=8, scaling="yarn", original=0), dict(rot_dim=8, scaling="yarn", slow=3.0, fast=2.0)):
        with pytest.raises(ValueError):
            ops.rope_frequencies(**kw)
    with pytest.raises(ValueError):
        ops.rope_plan(64, rot_dim=66)


def test_oracle_attention_of_known_weights():
    """One key of score 0 and one of ln 3: weights 1/4 and 3/4, the later token's alone."""
    q, v = np.array([[[1.0, 0.0]], [[1.0, 0.0]]]), np.array([[[4.0, 0.0]], [[0.0, 2.0]]])
    k = np.array([[[0.0, 3.0]], [[math.log(3.0), 5.0]]])
    out, bound = _prefill.attention(None, q, [0, 2], None, None, k, v, 1.0)
    assert np.allclose(out, [[[4.0, 0.0]], [[1.0, 1.5]]], rtol=1e-12) and (bound > 0).any()
    v[1, 0, 0] = np.inf
    out, _ = _prefill.attention(None, q, [0, 2], None, None, k, v, 1.0)
    assert np.array_equal(out[0], [[4.0, 0.0]]) and out[1, 0, 0] == np.inf and out[1, 0, 1] == 1.5


def test_heads_of_no_channels_are_refused():
    torch = pytest.importorskip("torch")
    from longhornai_amd import ops
    x, offs = torch.zeros((3, 8), dtype=torch.int16), torch.zeros(2, dtype=torch.int32)
    for D in (0, -8):
        with pytest.raises(ValueError, match="head_dim"):
            ops.attn_prompt(x, x, x, offs, D)
        with pytest.raises(ValueError, match="head_dim"):
            ops.rope_plan(D, rot_dim=0)


@pytest.mark.parametrize("kw,code", [
    (dict(seqs=-1), INV), (dict(cap=-1), INV), (dict(width=-1), INV), (dict(pages=-1), INV), (dict(width=1 << 25), UNS),
    (dict(cap=2 ** 31 - 1), UNS), (dict(seqs=2 ** 31 - 1), UNS), (dict(lengths=None), INV), (dict(left=None), INV),
    (dict(table=None), INV), (dict(owned=None), INV)])
def test_plan_with_owned_pages_refusals(L, kw, code):
    a = dict(zip(("lengths", "new", "tree", "left", "left_out", "free", "table"), plan_args()[:7])) | dict(owned=FAKE) | \
        dict(zip(("offsets", "positions", "slots", "seqs", "cap", "width", "pages", "stream"), plan_args()[7:]))
    a.update(kw)
    assert L.status("lhq_kv_plan_owned", *a.values()) == code, L.last_error()
    assert "kv_plan_owned" in L.last_error()


def test_plan_helper_refuses_counts_of_another_kind():
    i32 = dict(dtype=torch.int32)
    for owned in (torch.zeros(3, **i32), torch.zeros(2, dtype=torch.int64), torch.zeros(4, **i32)[::2], torch.zeros((2, 1), **i32)):
        with pytest.raises(ValueError, match="owned"):
            ops.kv_plan(torch.zeros(2, **i32), torch.ones(2, **i32), torch.zeros(5, **i32), torch.zeros(2, **i32),
                        torch.zeros((2, 3), **i32), 2, owned=owned)


# 5 rows of 32 heads of 128 from `out` on, in bytes
OUT, OUT_BYTES = 8 << 20, 5 * 4096 * 2


@pytest.mark.parametrize("fn,args", [("lhq_attn_prompt_bf16", prompt_args), ("lhq_kv_prefill_bf16", prefill_args)])
@pytest.mark.parametrize("kw", [
    dict(k=OUT), dict(v=OUT), dict(k=OUT + OUT_BYTES - 2), dict(v=OUT - 5 * 1024 * 2 + 2), dict(q=OUT - 2), dict(q=OUT + 4096 * 2),
    dict(q=OUT, qs=4104), dict(q=OUT + OUT_BYTES - 2), dict(q=OUT - OUT_BYTES + 2),
    dict(k=OUT - 4 * 30000 * 2 - 2046, ks=30000),          # the last row's last element
    dict(v=OUT - 3 * 30000 * 2 + OUT_BYTES - 2, vs=30000),  # a row in the middle
])
def test_results_over_what_others_read_are_refused(L, fn, args, kw):
    """Workgroups read keys and values in no order with the writing of results."""
    at = dict(q=16 << 20, k=24 << 20, v=32 << 20, out=OUT) | kw
    assert L.status(fn, *args(**{n: C.c_void_p(x) if n in ("q", "k", "v", "out") else x for n, x in at.items()})) == INV
    assert "overlap" in L.last_error()


def test_assembly_names_the_registers_it_writes():
    """A statement that sets m0 says so, else the compiler may keep something there."""
    import glob
    import os
    import re
    sources = glob.glob(os.path.join(os.path.dirname(os.path.abspath(capi.__file__)), "csrc", "*.h*"))
    found = 0
    for path in sources:
        for text in re.findall(r"asm\s+volatile\s*\((.*?)\)\s*;", open(path).read(), flags=re.S):
            if re.search(r"\b[sv]_\w+\s+m0\s*,", text):
                found += 1
                assert '"m0"' in text.rsplit(":", 1)[1], (path, text)
    assert found >= 2


def test_the_middle_of_the_yarn_ramp_is_by_turns():
    """Worked out by hand.  theta 10000 and 4 channels: 1 and 0.01 radians a position; in 4096
    positions the second makes 4096 * 0.01 / (2 pi) = 6.518986469 turns, (6.518986469 - 1) / 31 =
    0.178031822 of the way from 1 turn to 32: 0.0025 * 0.821968178 + 0.01 * 0.178031822."""
    f = ops.rope_frequencies(4, theta=10000.0, scaling="yarn", factor=4.0, original=4096)
    assert f[0] == 1.0 and math.isclose(f[1], 0.003835238663, rel_tol=1e-9)
    # theta 16, original 64: 1, 1/2, 1/4 and 1/8 make 64 / (2 pi) = 10.18591635788 turns, 5.09295817894,
    # 2.54647908947 and 1.273...; from 2 to 6 that is 1, 3.09295817894 / 4 = 0.773239544735,
    # 0.54647908947 / 4 = 0.136619772368 and 0 of the way k, and (1 + k) / 2 of each frequency
    f = ops.rope_frequencies(8, theta=16.0, scaling="yarn", factor=2.0, original=64, slow=2.0, fast=6.0)
    assert np.allclose(f, [1.0, 0.25 * 1.773239544735, 0.125 * 1.136619772368, 0.0625], rtol=1e-9, atol=0)


def test_plans_of_given_frequencies(monkeypatch):
    monkeypatch.setattr(ops, "dev", torch.from_numpy)
    f = ops.rope_frequencies(64, theta=500000.0, scaling="yarn", factor=4.0)
    a = ops.rope_plan(128, 64, theta=500000.0, scaling="yarn", factor=4.0)
    b = ops.rope_plan(128, 64, frequencies=f, gain=a.gain)
    assert torch.equal(a.turns, b.turns) and (a.rot_dim, a.gain) == (b.rot_dim, b.gain)
    assert ops.rope_plan(128, 64, frequencies=f).gain == 1.0
    # a quarter turn, the same backwards, one and a quarter, none, nearly none backwards
    quarter = np.pi / 2
    turns = ops.rope_plan(10, frequencies=np.array([quarter, -quarter, 5 * quarter, 0.0, -1e-300])).turns
    assert turns.numpy().view(np.uint64).tolist() == [1 << 62, 3 << 62, 1 << 62, 0, 0]
    for kw in (dict(frequencies=f[:31]), dict(frequencies=f[None]), dict(frequencies=np.where(f < 1, f, np.nan)),
               dict(frequencies=np.where(f < 1, f, np.inf)), dict(frequencies=f, scaling="linear"), dict(frequencies=[])):
        with pytest.raises(ValueError, match="frequencies"):
            ops.rope_plan(128, 64, **kw)
    with pytest.raises(ValueError):
        ops.rope_plan(128, 63, frequencies=f[:31])
