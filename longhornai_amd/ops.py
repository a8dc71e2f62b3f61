"""Torch-tensor helpers over the C ABI, for tests and ``bench.py``.

Torch is only plumbing here: it owns device memory and the current stream.
Every compute call goes through ``liblonghorn_hip.so`` (``capi.load()``), and
a missing library raises -- nothing here computes anything itself.

bf16 / fp16 data travels as raw 16-bit patterns in ``torch.int16`` tensors so
no torch conversion can touch the bits.
"""
from __future__ import annotations

from dataclasses import dataclass

import numpy as np
import torch

from . import capi

_NP_TO_TORCH = {
    np.dtype(np.float32): torch.float32,
    np.dtype(np.int8): torch.int8,
    np.dtype(np.uint8): torch.uint8,
    np.dtype(np.int16): torch.int16,
    np.dtype(np.int32): torch.int32,
    np.dtype(np.int64): torch.int64,
}
_VIEW = {np.dtype(np.uint16): np.int16, np.dtype(np.uint32): np.int32}


def lib():
    return capi.load()


# The current stream's handle straight from the runtime binding:
# torch.cuda.current_stream() builds a Stream object for it, 2.8 us of an 8 us
# decode call against 0.3.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def stream() -> int:
    if _raw_stream is None:
        return torch.cuda.current_stream().cuda_stream
    return _raw_stream(torch.cuda.current_device())


def dev(a: np.ndarray, device: str = "cuda") -> torch.Tensor:
    """Copy a numpy array to the device, bit for bit (uint16/uint32 via int views)."""
    a = np.ascontiguousarray(a)
    if a.dtype in _VIEW:
        a = a.view(_VIEW[a.dtype])
    return torch.from_numpy(a.copy()).to(device)


def host(t: torch.Tensor, dtype=None) -> np.ndarray:
    a = t.detach().cpu().numpy()
    return a.view(dtype) if dtype is not None else a


def empty(shape, np_dtype, device: str = "cuda") -> torch.Tensor:
    dt = np.dtype(np_dtype)
    dt = np.dtype(_VIEW.get(dt, dt))
    return torch.empty(tuple(shape), dtype=_NP_TO_TORCH[dt], device=device)


def zeros(shape, np_dtype, device: str = "cuda") -> torch.Tensor:
    t = empty(shape, np_dtype, device)
    t.zero_()
    return t


def P(t) -> int:
    return 0 if t is None else t.data_ptr()


def run(name: str, *args) -> None:
    """Call a C-ABI entry point with tensors passed directly.

    Tensors (and numpy arrays, copied to the device here) stay referenced
    until the call has enqueued its kernels; after that, torch's
    stream-ordered allocator cannot hand their memory to later work on the
    same stream before the kernels finish."""
    keep = []  # copies made here (the caller's tensors are held by args)
    conv = []
    for a in args:
        if isinstance(a, torch.Tensor):
            conv.append(a.data_ptr())
        elif a is None:
            conv.append(0)
        elif isinstance(a, np.ndarray):
            a = dev(a)
            keep.append(a)
            conv.append(a.data_ptr())
        else:
            conv.append(a)
    lib().call(name, *conv, stream())
    del keep


# ---------------------------------------------------------------------------
# Prepacked weights
# ---------------------------------------------------------------------------

@dataclass
class W4Weights:
    """Prepacked int4 weights (layout in include/longhorn_hip.h)."""
    qweight: torch.Tensor
    scales: torch.Tensor
    zeros: torch.Tensor | None
    K: int
    N: int
    G: int
    asym: bool

    @property
    def nbytes(self) -> int:
        n = self.qweight.numel() + self.scales.numel() * self.scales.element_size()
        if self.zeros is not None:
            n += self.zeros.numel() * 4
        return n


def w4_buffers(K: int, N: int, G: int, asym: bool):
    L = lib()
    qb = L.lhq_w4_qweight_bytes(K, N)
    sb = L.lhq_w4_scales_bytes(K, N, G, 1 if asym else 0)
    zb = L.lhq_w4_zeros_bytes(K, N, G) if asym else 0
    if qb <= 0 or sb <= 0:
        raise ValueError(f"bad W4 dims K={K} N={N} G={G}")
    q = empty((qb,), np.uint8)
    s = empty((sb // 2,), np.int16) if asym else empty((sb // 4,), np.float32)
    z = empty((zb // 4,), np.int32) if asym else None
    return q, s, z


def prepack_w4_sym(packed: torch.Tensor, scales: torch.Tensor, K: int, N: int, G: int) -> W4Weights:
    """Reference-layout int4 ([K/2,N] bytes, fp32 [K/G,N] scales) -> prepacked."""
    q, s, _ = w4_buffers(K, N, G, False)
    lib().call("lhq_w4_prepack_sym", P(packed), P(scales), K, N, G, P(q), P(s), stream())
    return W4Weights(q, s, None, K, N, G, False)


def prepack_w4_asym(packed: torch.Tensor, scales_f16: torch.Tensor, zeros_u8: torch.Tensor,
                    K: int, N: int, G: int) -> W4Weights:
    q, s, z = w4_buffers(K, N, G, True)
    lib().call("lhq_w4_prepack_asym", P(packed), P(scales_f16), P(zeros_u8), K, N, G,
               P(q), P(s), P(z), stream())
    return W4Weights(q, s, z, K, N, G, True)


def interleave_gate_up(wg: W4Weights, wu: W4Weights) -> W4Weights:
    """Gate and up projections [K, I] (asymmetric, prepacked) -> one tensor
    with 2 ceil(I/16) interleaved column tiles; N stays I."""
    if (wg.K, wg.N, wg.G, wg.asym) != (wu.K, wu.N, wu.G, wu.asym) or not wg.asym:
        raise ValueError("gate and up must be asymmetric W4 of one shape")
    q = empty((2 * wg.qweight.numel(),), np.uint8)
    s = empty((2 * wg.scales.numel(),), np.int16)
    z = empty((2 * wg.zeros.numel(),), np.int32)
    lib().call("lhq_w4_interleave_gate_up", P(wg.qweight), P(wg.scales), P(wg.zeros), P(wu.qweight),
               P(wu.scales), P(wu.zeros), wg.K, wg.N, wg.G, P(q), P(s), P(z), stream())
    return W4Weights(q, s, z, wg.K, wg.N, wg.G, True)


def pointer_tables(ws: list[W4Weights]):
    """Device arrays of the per-group qweight / scales / zeros pointers."""
    def tab(ts):
        return torch.tensor([t.data_ptr() for t in ts], dtype=torch.int64, device="cuda")
    return tab([w.qweight for w in ws]), tab([w.scales for w in ws]), tab([w.zeros for w in ws])


def prepack_b8(B: torch.Tensor, K: int, N: int) -> torch.Tensor:
    nbytes = lib().lhq_b8_prepacked_bytes(K, N)
    Bt = empty((nbytes,), np.uint8)
    lib().call("lhq_b8_prepack", P(B), K, N, P(Bt), stream())
    return Bt


# ---------------------------------------------------------------------------
# GEMMs
# ---------------------------------------------------------------------------

def gemm_w4a16(A: torch.Tensor, w: W4Weights, C: torch.Tensor | None = None,
               alpha: float = 1.0, beta: float = 0.0) -> torch.Tensor:
    """fp32 A [M,K], symmetric weights, fp32 C (reference semantics)."""
    M = A.shape[0]
    if C is None:
        C = zeros((M, w.N), np.float32)
    lib().call("lhq_gemm_w4a16", P(A), P(w.qweight), P(w.scales), P(C), M, w.N, w.K, w.G,
               alpha, beta, stream())
    return C


def w4a16_bf16_workspace(M: int, w: W4Weights) -> torch.Tensor | None:
    """A device workspace of the size lhq_gemm_w4a16_bf16_ws asks for (None
    when the shape runs without one)."""
    n = lib().lhq_gemm_w4a16_bf16_workspace_bytes(M, w.N, w.K, w.G)
    return empty((n,), np.uint8) if n > 0 else None


def gemm_w4a16_bf16_ws(A: torch.Tensor, w: W4Weights, ws: torch.Tensor | None,
                       C: torch.Tensor | None = None) -> torch.Tensor:
    """gemm_w4a16_bf16 with a workspace (K split across workgroups where the
    output grid is thin)."""
    M = A.shape[0]
    if C is None:
        C = empty((M, w.N), np.int16)
    nbytes = 0 if ws is None else ws.numel() * ws.element_size()
    lib().call("lhq_gemm_w4a16_bf16_ws", P(A), P(w.qweight), P(w.scales), P(w.zeros), P(C),
               M, w.N, w.K, w.G, P(ws), nbytes, stream())
    return C


def gemm_w4a16_bf16_noalloc(A: torch.Tensor, w: W4Weights, C: torch.Tensor) -> torch.Tensor:
    """gemm_w4a16_bf16_ws on the library's static scratch: allocates nothing."""
    M = A.shape[0]
    lib().call("lhq_gemm_w4a16_bf16_noalloc", P(A), P(w.qweight), P(w.scales), P(w.zeros), P(C),
               M, w.N, w.K, w.G, stream())
    return C


def gemm_w4a16_bf16(A: torch.Tensor, w: W4Weights, C: torch.Tensor | None = None) -> torch.Tensor:
    """bf16 A [M,K] (int16 bits), asymmetric weights, bf16 C [M,N] (int16 bits)."""
    M = A.shape[0]
    if C is None:
        C = empty((M, w.N), np.int16)
    lib().call("lhq_gemm_w4a16_bf16", P(A), P(w.qweight), P(w.scales), P(w.zeros), P(C),
               M, w.N, w.K, w.G, stream())
    return C


def gemm_w8a8(Aq, Bt, As, Bs, M, N, K, C=None, alpha=1.0, beta=0.0):
    if C is None:
        C = zeros((M, N), np.float32)
    lib().call("lhq_gemm_w8a8", P(Aq), P(Bt), P(As), P(Bs), P(C), M, N, K, alpha, beta, stream())
    return C


def gemm_w8a8_bf16(Aq, Bt, As, Bs, M, N, K, C=None):
    if C is None:
        C = empty((M, N), np.int16)
    lib().call("lhq_gemm_w8a8_bf16", P(Aq), P(Bt), P(As), P(Bs), P(C), M, N, K, stream())
    return C


def gemm_w8a8_i32(Aq, Bt, M, N, K, C=None):
    if C is None:
        C = empty((M, N), np.int32)
    lib().call("lhq_gemm_w8a8_i32", P(Aq), P(Bt), P(C), M, N, K, stream())
    return C


# ---------------------------------------------------------------------------
# 8-bit key/value cache and attention over it
# ---------------------------------------------------------------------------

KV_PAGE = 64
KV_MAX_NEW = 64  # new tokens of one sequence that a call of kv_attn attends
_KV_FORMATS = {"int8": 0, "fp8": 1}  # LHQ_KV_INT8, LHQ_KV_FP8


@dataclass(frozen=True)
class KvCache:
    """The buffers of a paged 8-bit cache (layout in include/longhorn_hip.h):
    codes uint8 (keys [pages, heads, 64, Dp], values [pages, heads, Dp, 64]),
    scales fp32 [pages, heads, 64].  ``fmt`` is "int8" or "fp8"."""
    fmt: str
    n_pages: int
    n_kv_heads: int
    head_dim: int
    k: torch.Tensor
    v: torch.Tensor
    k_scales: torch.Tensor
    v_scales: torch.Tensor

    def __post_init__(self):
        if self.fmt not in _KV_FORMATS:
            raise ValueError(f"KvCache: format {self.fmt!r} is not one of {sorted(_KV_FORMATS)}")
        L, dims = lib(), (self.n_pages, self.n_kv_heads, self.head_dim)
        codes, scales = L.lhq_kv_codes_bytes(*dims), L.lhq_kv_scales_bytes(*dims[:2])
        if codes <= 0 or scales <= 0:
            raise ValueError(f"KvCache: bad dims pages={dims[0]} heads={dims[1]} head_dim={dims[2]}")
        for name, t, dt, nbytes in (("k", self.k, torch.uint8, codes), ("v", self.v, torch.uint8, codes),
                                    ("k_scales", self.k_scales, torch.float32, scales),
                                    ("v_scales", self.v_scales, torch.float32, scales)):
            if t.dtype != dt or not t.is_contiguous() or t.numel() * t.element_size() != nbytes:
                raise ValueError(f"KvCache: {name} must be {nbytes} contiguous bytes of {dt}, "
                                 f"got {tuple(t.shape)} {t.dtype}")
            if t.device != self.k.device:
                raise ValueError(f"KvCache: {name} is on {t.device}, k on {self.k.device}")

    def pointers(self):
        return self.k.data_ptr(), self.k_scales.data_ptr(), self.v.data_ptr(), self.v_scales.data_ptr()


def kv_cache(fmt: str, n_pages: int, n_kv_heads: int, head_dim: int) -> KvCache:
    """A cache of its own memory; its tokens hold nothing until they are written."""
    L = lib()
    codes, scales = L.lhq_kv_codes_bytes(n_pages, n_kv_heads, head_dim), L.lhq_kv_scales_bytes(n_pages, n_kv_heads)
    if codes <= 0 or scales <= 0:
        raise ValueError(f"kv_cache: bad dims pages={n_pages} heads={n_kv_heads} head_dim={head_dim}")
    return KvCache(fmt, n_pages, n_kv_heads, head_dim, zeros((codes,), np.uint8), zeros((codes,), np.uint8),
                   zeros((scales // 4,), np.float32), zeros((scales // 4,), np.float32))


# These checks run before every call, ahead of kernels of a few microseconds:
# each attribute of a tensor is read once, the usual case decided first.

def _kv_on_gpu(fn: str, cache: KvCache, *tensors: torch.Tensor | None) -> None:
    """The cache and what goes with it lie on one GPU: the kernels fault on other
    addresses (0.1 us a tensor)."""
    at = cache.k.get_device()
    if at < 0:
        raise ValueError(f"{fn}: the cache is not on a GPU")
    for t in tensors:
        if t is not None and t.get_device() != at:
            raise ValueError(f"{fn}: a tensor of {t.device} with a cache on GPU {at}")


def _kv_rows(fn: str, name: str, t: torch.Tensor, heads: int, D: int, dtypes) -> tuple[int, int]:
    """Checks new tokens' rows [n, heads * D] or [n, heads, D], heads packed;
    returns (rows, the stride between them)."""
    shape, st = t.shape, t.stride()
    if t.dtype not in dtypes:
        raise ValueError(f"{fn}: {name} is {t.dtype}, not one of {[str(d) for d in dtypes]}")
    width = heads * D
    if len(shape) == 2 and shape[1] == width:
        packed = st[1] == 1 or width == 1
    elif len(shape) == 3 and shape[1] == heads and shape[2] == D:
        packed = (st[2] == 1 or D == 1) and (st[1] == D or heads == 1)
    else:
        raise ValueError(f"{fn}: {name} has shape {tuple(shape)}, not [n, {heads} * {D}]")
    if not packed:
        raise ValueError(f"{fn}: the heads of a row of {name} must lie one after the other (strides {tuple(st)})")
    n = shape[0]
    return n, st[0] if n > 1 else max(st[0], width)


def _kv_tables(fn: str, offsets: torch.Tensor, start: torch.Tensor, table: torch.Tensor):
    """Checks the int32 device tables; returns (sequences, pages of a table row)."""
    i32 = torch.int32
    if offsets.dtype is not i32 or start.dtype is not i32 or table.dtype is not i32:
        raise ValueError(f"{fn}: offsets, positions and block table must be int32")
    positions, offs, shape = start.shape, offsets.shape, table.shape
    if len(positions) != 1 or len(offs) != 1 or len(shape) != 2 or offs[0] != positions[0] + 1 or shape[0] != positions[0]:
        raise ValueError(f"{fn}: positions {tuple(positions)}, offsets {tuple(offs)} and block table {tuple(shape)} are "
                         "not [B], [B + 1] and [B, pages]")
    if not (offsets.is_contiguous() and start.is_contiguous() and table.is_contiguous()):
        raise ValueError(f"{fn}: offsets, positions and block table must be contiguous")
    return positions[0], shape[1]


_KV_BITS, _KV_ROWS = (torch.int16,), (torch.int16, torch.float32)


def kv_write(cache: KvCache, k: torch.Tensor, v: torch.Tensor, offsets: torch.Tensor, start: torch.Tensor,
             block_table: torch.Tensor, rows: torch.Tensor | None = None) -> None:
    """Quantize new tokens into the cache.  k, v: fp32, or bf16 as int16 bits,
    [n, heads * head_dim] (rows may be strided); sequence s's rows
    offsets[s] .. offsets[s+1] go to its positions from start[s] on.  ``rows``
    (int32): the row of k and v for each row of that list (one outside them is
    skipped)."""
    H, D = cache.n_kv_heads, cache.head_dim
    dt = k.dtype
    n_rows, ks = _kv_rows("kv_write", "k", k, H, D, _KV_ROWS)
    n_values, vs = _kv_rows("kv_write", "v", v, H, D, (dt,))
    B, width = _kv_tables("kv_write", offsets, start, block_table)
    if n_values != n_rows:
        raise ValueError(f"kv_write: {n_rows} rows of keys and {n_values} of values")
    if rows is not None and (rows.dtype != torch.int32 or not rows.is_contiguous()):
        raise ValueError("kv_write: rows must be contiguous int32")
    _kv_on_gpu("kv_write", cache, k, v, offsets, start, block_table, rows)
    n = n_rows if rows is None else rows.numel()
    lib().call("lhq_kv_write_f32" if dt == torch.float32 else "lhq_kv_write_bf16", k.data_ptr(), v.data_ptr(), ks, vs,
               P(rows), offsets.data_ptr(), start.data_ptr(), block_table.data_ptr(), *cache.pointers(),
               _KV_FORMATS[cache.fmt], B, n_rows, n, width, cache.n_pages, H, D, stream())


def kv_read(cache: KvCache, offsets: torch.Tensor, start: torch.Tensor, block_table: torch.Tensor, n: int,
            bf16: bool = True, out: tuple[torch.Tensor, torch.Tensor] | None = None):
    """Cached tokens as values: row i of sequence s's rows offsets[s] ..
    offsets[s+1] is its position start[s] + i.  n rows in all; returns (k, v)
    [n, heads, head_dim], bf16 as int16 bits or fp32.  Rows that offsets give to
    no sequence are not written."""
    H, D = cache.n_kv_heads, cache.head_dim
    B, width = _kv_tables("kv_read", offsets, start, block_table)
    dt = torch.int16 if bf16 else torch.float32
    if out is None:
        k = cache.k.new_empty((n, H, D), dtype=dt)
        out = k, torch.empty_like(k)
    else:
        for t in out:
            if t.dtype != dt or tuple(t.shape) != (n, H, D) or not t.is_contiguous():
                raise ValueError(f"kv_read: outputs must be contiguous [{n}, {H}, {D}] {dt}")
    _kv_on_gpu("kv_read", cache, offsets, start, block_table, *out)
    lib().call("lhq_kv_read_bf16" if bf16 else "lhq_kv_read_f32", *cache.pointers(), offsets.data_ptr(),
               start.data_ptr(), block_table.data_ptr(), out[0].data_ptr(), out[1].data_ptr(),
               _KV_FORMATS[cache.fmt], B, n, width, cache.n_pages, H, D, stream())
    return out


def kv_attn_workspace(cache: KvCache, n_seqs: int, n: int, max_new: int, max_pages: int,
                      n_heads: int) -> torch.Tensor | None:
    """A device workspace of the size lhq_kv_attn_bf16 can use (None: it needs none)."""
    nbytes = lib().lhq_kv_attn_workspace_bytes(n_seqs, n, max_new, max_pages, n_heads, cache.n_kv_heads,
                                               cache.head_dim)
    return empty((nbytes,), np.uint8) if nbytes > 0 else None


def kv_attn(cache: KvCache, q: torch.Tensor, offsets: torch.Tensor, lengths: torch.Tensor,
            block_table: torch.Tensor, k_new: torch.Tensor | None, v_new: torch.Tensor | None,
            tree: torch.Tensor | None = None, scale: float | None = None, max_new: int | None = None,
            workspace: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of new tokens (q [n, heads * head_dim], bf16 as int16 bits)
    over the first lengths[s] cached tokens of their sequence and over the new
    ones (k_new, v_new) that tree (int64, a bit for each) names -- None: those
    up to the token itself.  Returns out [n, heads, head_dim], int16 bits.
    max_new bounds the new tokens of one sequence, 64 at most; the closer, the
    better the kernel's shape (1 in plain decode).  Rows past it in a sequence,
    and rows of q that offsets give to none, are not computed: they stay what
    ``out`` held.  None: as many as q has rows, 64 at most, and what is not
    computed is zero in a result that is made here."""
    H, D = cache.n_kv_heads, cache.head_dim
    B, width = _kv_tables("kv_attn", offsets, lengths, block_table)
    shape = q.shape
    heads = shape[1] // D if len(shape) == 2 else shape[1] if len(shape) == 3 else 0
    n, qs = _kv_rows("kv_attn", "q", q, heads, D, _KV_BITS)
    if heads % H != 0:
        raise ValueError(f"kv_attn: {heads} query heads over {H} kv heads")
    if (k_new is None) != (v_new is None):
        raise ValueError("kv_attn: new keys without values, or values without keys")
    ks = vs = 0
    if k_new is not None:
        n_keys, ks = _kv_rows("kv_attn", "k_new", k_new, H, D, _KV_BITS)
        n_values, vs = _kv_rows("kv_attn", "v_new", v_new, H, D, _KV_BITS)
        if n_keys != n or n_values != n:
            raise ValueError(f"kv_attn: {n} queries with {n_keys} new keys and {n_values} values")
    if tree is not None and (tree.dtype != torch.int64 or tree.numel() != n or not tree.is_contiguous()):
        raise ValueError(f"kv_attn: tree must hold {n} contiguous int64 words")
    bound = min(n, KV_MAX_NEW) if max_new is None else max_new
    if out is None:
        if max_new is not None and n > B * max_new:
            raise ValueError(f"kv_attn: {n} rows of {B} sequences are over max_new = {max_new} each, and no out is "
                             "given for those that are not computed")
        out = q.new_empty((n, heads, D)) if max_new is not None else q.new_zeros((n, heads, D))
    elif out.dtype != torch.int16 or out.numel() != n * heads * D or not out.is_contiguous():
        raise ValueError(f"kv_attn: out must be contiguous [{n}, {heads}, {D}] int16")
    nbytes = 0
    if workspace is not None:
        if not workspace.is_contiguous():
            raise ValueError(f"kv_attn: workspace must be contiguous (strides {tuple(workspace.stride())})")
        nbytes = workspace.numel() * workspace.element_size()
    _kv_on_gpu("kv_attn", cache, q, offsets, lengths, block_table, k_new, v_new, tree, workspace, out)
    lib().call("lhq_kv_attn_bf16", q.data_ptr(), qs, P(k_new), ks, P(v_new), vs, P(tree), offsets.data_ptr(),
               lengths.data_ptr(), block_table.data_ptr(), *cache.pointers(), out.data_ptr(), _KV_FORMATS[cache.fmt],
               B, n, bound, width, cache.n_pages, heads, H, D, D ** -0.5 if scale is None else scale, P(workspace),
               nbytes, stream())
    return out
