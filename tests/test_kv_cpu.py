"""The key/value cache without a GPU: sizes, refusals of the C ABI and of the
Python helpers, and the layout's definition."""
import ctypes as C

import numpy as np
import pytest
import torch

from longhornai_amd import capi, ops
from tests import _kv

FAKE = C.c_void_p(0x1000)  # never dereferenced: validation fails first
ODD = C.c_void_p(0x1004)
INV, UNS = capi.LHQ_ERR_INVALID, capi.LHQ_ERR_UNSUPPORTED


@pytest.fixture(scope="module")
def L():
    return capi.load()


def test_sizes(L):
    assert L.lhq_kv_codes_bytes(10, 8, 128) == 10 * 8 * 64 * 128
    assert L.lhq_kv_codes_bytes(3, 5, 75) == 3 * 5 * 64 * 96   # padded to 32 channels
    assert L.lhq_kv_codes_bytes(1 << 20, 16, 256) == 1 << 38    # past 32 bits
    assert L.lhq_kv_scales_bytes(10, 8) == 10 * 8 * 64 * 4
    for bad in ((-1, 8, 128), (4, 0, 128), (4, 8, 0), (4, 8, 257)):
        assert L.lhq_kv_codes_bytes(*bad) == 0
    assert L.lhq_kv_scales_bytes(-1, 8) == L.lhq_kv_scales_bytes(4, 0) == 0
    ws = L.lhq_kv_attn_workspace_bytes
    assert ws(4, 4, 1, 100, 32, 8, 128) >= 0
    for bad in ((-1, 4, 1, 9, 8, 8, 64), (4, -1, 1, 9, 8, 8, 64), (4, 4, 65, 9, 8, 8, 64), (4, 4, 1, -1, 8, 8, 64),
                (4, 4, 1, 9, 9, 8, 64), (4, 4, 1, 9, 8, 0, 64), (4, 4, 1, 9, 8, 8, 300)):
        assert ws(*bad) == 0


def test_value_rows_hold_every_token_once():
    assert sorted(_kv.SLOTS) == list(range(64))


def write_args(**kw):
    a = dict(k=FAKE, v=FAKE, ks=1024, vs=1024, rows=None, offsets=FAKE, start=FAKE, table=FAKE, kc=FAKE, ksc=FAKE,
             vc=FAKE, vsc=FAKE, fmt=0, seqs=2, n_rows=5, cap=5, width=4, pages=9, heads=8, D=128, stream=None)
    a.update(kw)
    return list(a.values())


def read_args(**kw):
    a = dict(kc=FAKE, ksc=FAKE, vc=FAKE, vsc=FAKE, offsets=FAKE, start=FAKE, table=FAKE, ko=FAKE, vo=FAKE, fmt=0,
             seqs=2, cap=5, width=4, pages=9, heads=8, D=128, stream=None)
    a.update(kw)
    return list(a.values())


def attn_args(**kw):
    a = dict(q=FAKE, qs=4096, k=FAKE, ks=1024, v=FAKE, vs=1024, tree=None, offsets=FAKE, lengths=FAKE, table=FAKE,
             kc=FAKE, ksc=FAKE, vc=FAKE, vsc=FAKE, out=FAKE, fmt=0, seqs=2, cap=5, max_new=4, width=4, pages=9,
             heads=32, kv=8, D=128, scale=0.1, ws=None, wsb=0, stream=None)
    a.update(kw)
    return list(a.values())


COMMON = [(dict(fmt=2), INV), (dict(fmt=-1), INV), (dict(seqs=-1), INV), (dict(cap=-1), INV), (dict(width=-1), INV),
          (dict(pages=-1), INV), (dict(D=0), INV), (dict(D=257), UNS), (dict(width=1 << 25), UNS),
          (dict(offsets=None), INV), (dict(table=None), INV), (dict(kc=None), INV), (dict(ksc=None), INV),
          (dict(vc=None), INV), (dict(vsc=None), INV), (dict(kc=ODD), INV), (dict(vc=ODD), INV), (dict(ksc=ODD), INV),
          (dict(vsc=ODD), INV)]


@pytest.mark.parametrize("kw,code", COMMON + [
    (dict(heads=0), INV), (dict(heads=70000, ks=1 << 40, vs=1 << 40), UNS), (dict(k=None), INV), (dict(v=None), INV),
    (dict(start=None), INV), (dict(n_rows=-1), INV), (dict(ks=1023), INV), (dict(vs=0), INV), (dict(ks=-1024), INV)])
@pytest.mark.parametrize("fn", ["lhq_kv_write_f32", "lhq_kv_write_bf16"])
def test_write_refusals(L, fn, kw, code):
    assert L.status(fn, *write_args(**kw)) == code, L.last_error()
    assert fn[4:] in L.last_error()


@pytest.mark.parametrize("kw,code", COMMON + [(dict(heads=0), INV), (dict(ko=None), INV), (dict(vo=None), INV),
                                              (dict(start=None), INV)])
@pytest.mark.parametrize("fn", ["lhq_kv_read_f32", "lhq_kv_read_bf16"])
def test_read_refusals(L, fn, kw, code):
    assert L.status(fn, *read_args(**kw)) == code, L.last_error()


@pytest.mark.parametrize("kw,code", COMMON + [
    (dict(kv=0), INV), (dict(heads=30), INV), (dict(heads=0), INV), (dict(heads=-8), INV), (dict(max_new=-1), INV),
    (dict(max_new=65), UNS), (dict(scale=0.0), INV), (dict(scale=-1.0), INV), (dict(scale=float("nan")), INV),
    (dict(scale=float("inf")), INV), (dict(k=None), INV), (dict(v=None), INV), (dict(qs=4095), INV),
    (dict(ks=1000), INV), (dict(vs=1000), INV), (dict(wsb=-1), INV), (dict(ws=ODD, wsb=1 << 20), INV),
    (dict(q=None), INV), (dict(out=None), INV), (dict(lengths=None), INV)])
def test_attn_refusals(L, kw, code):
    assert L.status("lhq_kv_attn_bf16", *attn_args(**kw)) == code, L.last_error()
    assert "kv_attn" in L.last_error()


def test_nothing_to_do_is_ok(L):
    for kw in (dict(seqs=0), dict(cap=0)):
        assert L.status("lhq_kv_write_bf16", *write_args(k=None, **kw)) == 0
        assert L.status("lhq_kv_read_f32", *read_args(ko=None, **kw)) == 0
        assert L.status("lhq_kv_attn_bf16", *attn_args(q=None, **kw)) == 0
    assert L.status("lhq_kv_write_f32", *write_args(n_rows=0, k=None)) == 0
    assert L.status("lhq_kv_attn_bf16", *attn_args(max_new=0, out=None)) == 0


def host_cache(**kw):
    c = _kv.HostCache("int8", 4, 2, 40)
    a = dict(fmt="int8", n_pages=4, n_kv_heads=2, head_dim=40, k=torch.from_numpy(c.k), v=torch.from_numpy(c.v),
             k_scales=torch.from_numpy(c.ks), v_scales=torch.from_numpy(c.vs))
    a.update(kw)
    return ops.KvCache(**a)


@pytest.mark.parametrize("kw", [dict(fmt="int4"), dict(head_dim=300), dict(n_pages=5), dict(n_kv_heads=0),
                                dict(k=torch.zeros(10, dtype=torch.uint8)),
                                dict(k_scales=torch.zeros((4, 2, 64), dtype=torch.float64)),
                                dict(v_scales=torch.zeros((4, 2, 128))[..., ::2])])
def test_cache_handle_refusals(kw):
    with pytest.raises(ValueError):
        host_cache(**kw)


def test_helper_refusals():
    """The Python helpers refuse what the C ABI cannot see (types, shapes, strides)."""
    c = host_cache()
    i32 = dict(dtype=torch.int32)
    k = torch.zeros((6, 80), dtype=torch.int16)
    offs, start, table = torch.tensor([0, 3, 6], **i32), torch.zeros(2, **i32), torch.zeros((2, 2), **i32)
    q = torch.zeros((6, 160), dtype=torch.int16)
    bad_rows = [k[:, :79], k.to(torch.float64), torch.zeros((6, 160), dtype=torch.int16)[:, ::2],
                torch.zeros((6, 40, 2), dtype=torch.int16).transpose(1, 2), k.view(torch.uint8)]
    for x in bad_rows:
        with pytest.raises(ValueError):
            ops.kv_write(c, x, k, offs, start, table)
        with pytest.raises(ValueError):
            ops.kv_write(c, k, x, offs, start, table)
        with pytest.raises(ValueError):
            ops.kv_attn(c, q, offs, start, table, x, k)
    for t in ((offs.long(), start, table), (offs[:2], start, table), (offs, start, table[:1]), (offs, start, table[0]),
              (offs, start, torch.zeros((2, 4), **i32)[:, ::2])):
        with pytest.raises(ValueError):
            ops.kv_write(c, k, k, *t)
        with pytest.raises(ValueError):
            ops.kv_read(c, *t, 6)
        with pytest.raises(ValueError):
            ops.kv_attn(c, q, *t, k, k)
    with pytest.raises(ValueError):
        ops.kv_write(c, k, k[:5], offs, start, table)
    with pytest.raises(ValueError):
        ops.kv_write(c, k, k, offs, start, table, rows=torch.zeros(6, dtype=torch.int64))
    with pytest.raises(ValueError):
        ops.kv_read(c, offs, start, table, 6, out=(torch.zeros((6, 2, 40)), torch.zeros((6, 2, 40))))
    for tree in (torch.zeros(5, dtype=torch.int64), torch.zeros(6, dtype=torch.int32)):
        with pytest.raises(ValueError):
            ops.kv_attn(c, q, offs, start, table, k, k, tree=tree)
    with pytest.raises(ValueError):
        ops.kv_attn(c, q, offs, start, table, k[:5], k)
    with pytest.raises(ValueError):
        ops.kv_attn(c, q, offs, start, table, k, k, out=torch.zeros((6, 4, 40)))
    with pytest.raises(ValueError):  # values without keys
        ops.kv_attn(c, q, offs, start, table, None, k)
    with pytest.raises(ValueError):  # 3 query heads over 2 kv heads
        ops.kv_attn(c, q[:, :120], offs, start, table, k, k)


def test_oracle_attention_of_known_weights():
    """The tests' oracle on a case by hand: one key of score 0 and one of ln 3
    give the weights 1/4 and 3/4."""
    c = _kv.HostCache("int8", 1, 1, 2)
    c.put(0, 0, 0, [0, 0], [8, 0], 1.0, 0.5)
    out, bound = _kv.attention(c, np.array([[[1.0, 0.0]]]), [0, 1], [1], np.array([[0]], np.int32),
                               np.array([[[np.log(3.0), 5.0]]]), np.array([[[0.0, 2.0]]]), None, 1.0)
    assert np.allclose(out, [[[1.0, 1.5]]], rtol=1e-12) and (bound > 0).all()
