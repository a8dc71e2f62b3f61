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


# ---------------------------------------------------------------------------
# A prompt's way through an attention layer
# ---------------------------------------------------------------------------

@dataclass(frozen=True)
class KvPlan:
    """A step's tables (lhq_kv_plan): offsets int32 [B + 1], positions int32 [n],
    slots int64 [n], left int32 [2] (pages left, pages missing)."""
    offsets: torch.Tensor
    positions: torch.Tensor
    slots: torch.Tensor
    left: torch.Tensor


def _on_one_gpu(fn: str, first: torch.Tensor, *tensors: torch.Tensor | None) -> None:
    """All of them on the current GPU, on whose stream the call is launched."""
    at = first.get_device()
    if at < 0:
        raise ValueError(f"{fn}: a tensor is on {first.device}, not on a GPU")
    if at != torch.cuda.current_device():
        raise ValueError(f"{fn}: a tensor of {first.device}, the current GPU is {torch.cuda.current_device()}")
    for t in tensors:
        if t is not None and t.get_device() != at:
            raise ValueError(f"{fn}: a tensor of {t.device} with one of {first.device}")


def _packed(fn: str, name: str, t: torch.Tensor, dtype, shape) -> None:
    if t.dtype is not dtype or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{fn}: {name} must be contiguous {list(shape)} {dtype}, got {tuple(t.shape)} {t.dtype}")


def kv_plan(lengths: torch.Tensor, new_tokens: torch.Tensor, free_pages: torch.Tensor, left: torch.Tensor,
            block_table: torch.Tensor, n: int, tree: torch.Tensor | None = None,
            out: KvPlan | None = None, owned: torch.Tensor | None = None) -> KvPlan:
    """A step's tables from the requests' lengths (int32 [B]): sequence s holds
    lengths[s] tokens and gets new_tokens[s] more, or is over where that is
    negative.  Pages go back to and come off the stack ``free_pages`` (int32, one
    entry for each page there is), whose first left[0] entries count; block_table
    [B, pages] gets the new ones.  n: rows there are room for.  tree (int64 [n]):
    drafted tokens' ancestors, for their positions.  ``out`` may hold ``left``
    itself, for tables that live from step to step.  owned (int32 [B], zeros at first,
    kept from step to step): how many entries of its row a sequence has pages in, so that
    new tokens may be rejected, come again after pages ran out, or never be taken, and a
    request may stay over.  Without it a sequence has the pages of its lengths alone, which must
    then grow by all its new tokens, and become 0 once it is over, or pages are lost or
    go back twice."""
    i32, shape = torch.int32, block_table.shape
    if len(shape) != 2 or n < 0:
        raise ValueError(f"kv_plan: block table {tuple(shape)} is not [B, pages], or {n} rows")
    B, width = shape
    _packed("kv_plan", "block_table", block_table, i32, (B, width))
    _packed("kv_plan", "lengths", lengths, i32, (B,))
    _packed("kv_plan", "new_tokens", new_tokens, i32, (B,))
    _packed("kv_plan", "left", left, i32, (2,))
    if free_pages.dtype is not i32 or len(free_pages.shape) != 1 or not free_pages.is_contiguous():
        raise ValueError(f"kv_plan: free_pages must be contiguous [pages] int32, got {tuple(free_pages.shape)}")
    if tree is not None:
        _packed("kv_plan", "tree", tree, torch.int64, (n,))
    if owned is not None:
        _packed("kv_plan", "owned", owned, i32, (B,))
    if out is None:
        out = KvPlan(lengths.new_empty(B + 1), lengths.new_empty(n), lengths.new_empty(n, dtype=torch.int64),
                     lengths.new_empty(2))
    else:
        _packed("kv_plan", "out.offsets", out.offsets, i32, (B + 1,))
        _packed("kv_plan", "out.positions", out.positions, i32, (n,))
        _packed("kv_plan", "out.slots", out.slots, torch.int64, (n,))
        _packed("kv_plan", "out.left", out.left, i32, (2,))
    _on_one_gpu("kv_plan", lengths, new_tokens, free_pages, left, block_table, tree, owned, out.offsets,
                out.positions, out.slots, out.left)
    lib().call("lhq_kv_plan" if owned is None else "lhq_kv_plan_owned", lengths.data_ptr(), new_tokens.data_ptr(), P(tree),
               left.data_ptr(), out.left.data_ptr(), free_pages.data_ptr(), block_table.data_ptr(),
               *(() if owned is None else (owned.data_ptr(),)), out.offsets.data_ptr(), out.positions.data_ptr(),
               out.slots.data_ptr(), B, n, width, free_pages.shape[0], stream())
    return out


@dataclass(frozen=True)
class RopePlan:
    """How heads are turned: for each pair of the first rot_dim channels the
    fraction of a full turn per position, in units of 2^-64 (as int64 bits)."""
    head_dim: int
    rot_dim: int
    turns: torch.Tensor
    interleaved: bool
    gain: float


def rope_frequencies(rot_dim: int, theta: float = 10000.0, scaling: str | None = None, factor: float = 1.0,
                     original: int = 4096, slow: float = 1.0, fast: float = 32.0) -> np.ndarray:
    """Radians per position of each pair, theta^(-2i / rot_dim), for contexts
    ``factor`` times the ``original`` length:
      "linear"  all divided by factor (positions interpolated)
      "ntk"     theta times factor^(rot_dim / (rot_dim - 2)): the slowest pair is
                divided by factor, the fastest kept
      "yarn"    pairs that make under ``slow`` turns in the original length divided
                by factor, those over ``fast`` kept, between them in proportion to
                the turns they make, as the method's paper has it.  Checkpoints made
                by its released code have a ramp in the pair's index, between
                rounded ends, which differs in the middle (by a factor of up to 2 or
                3): give rope_plan their own ``frequencies``"""
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError(f"rope_frequencies: scaling {scaling!r} is not None, 'linear', 'ntk' or 'yarn'")
    if rot_dim < 0 or rot_dim % 2 or not 1.0 <= theta < np.inf or not 1.0 <= factor < np.inf:
        raise ValueError(f"rope_frequencies: rot_dim {rot_dim}, theta {theta}, factor {factor}: an even number, and "
                         "finite ones of 1 or more, are wanted")
    if scaling == "ntk":
        if rot_dim == 2:
            raise ValueError("rope_frequencies: one pair alone has no slowest and fastest")
        theta = theta * factor ** (rot_dim / (rot_dim - 2)) if rot_dim else theta
    f = float(theta) ** (-np.arange(0, rot_dim, 2, dtype=np.float64) / max(rot_dim, 1))
    if scaling == "linear":
        f = f / factor
    if scaling == "yarn":
        if not (original > 0 and fast > slow):
            raise ValueError(f"rope_frequencies: original {original}, slow {slow}, fast {fast}")
        keep = np.clip((original * f / (2 * np.pi) - slow) / (fast - slow), 0.0, 1.0)
        f = f / factor * (1 - keep) + f * keep
    return f


def rope_plan(head_dim: int, rot_dim: int | None = None, theta: float = 10000.0, interleaved: bool = False,
              scaling: str | None = None, factor: float = 1.0, original: int = 4096, slow: float = 1.0,
              fast: float = 32.0, gain: float | None = None, frequencies: np.ndarray | None = None) -> RopePlan:
    """The plan that ``rope`` takes, made once (rope_frequencies says what the
    numbers are).  gain multiplies the turned channels; None: 0.1 ln(factor) + 1
    with "yarn", else 1.  frequencies: radians per position of each pair [rot_dim /
    2], any finite ones, in place of theta's and the scaling's."""
    rot = head_dim if rot_dim is None else rot_dim
    if head_dim < 1 or not 0 <= rot <= head_dim:
        raise ValueError(f"rope_plan: rot_dim {rot} is no part of head_dim {head_dim}")
    if frequencies is None:
        f = rope_frequencies(rot, theta, scaling, factor, original, slow, fast)
    else:
        f = np.asarray(frequencies, np.float64)
        if scaling is not None or f.shape != (rot // 2,) or rot % 2 or not np.isfinite(f).all():
            raise ValueError(f"rope_plan: frequencies {f.shape} are not finite ones of {rot} / 2 pairs, or there is "
                             f"scaling {scaling!r} beside them")
    # (whole turns per position change nothing; a fraction that rounds to one is none)
    turns = np.array([int(x * 2.0 ** 64) % 2 ** 64 for x in f / (2 * np.pi) % 1.0], np.uint64)
    if gain is None:
        gain = 0.1 * float(np.log(factor)) + 1.0 if scaling == "yarn" else 1.0
    return RopePlan(head_dim, rot, dev(turns.view(np.int64)), bool(interleaved), float(gain))


def rope(plan: RopePlan, q: torch.Tensor | None, k: torch.Tensor | None, positions: torch.Tensor,
         q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps: float = 1e-6,
         out: tuple[torch.Tensor | None, torch.Tensor | None] | None = None):
    """Queries and keys (fp32, or bf16 as int16 bits, [n, heads * head_dim] or [n,
    heads, head_dim], rows may be strided; either may be None) turned by their
    positions (int32 [n]; rows of negative ones are passed on as they are), each
    head RMS-normed first where a weight [head_dim] is given.  Returns (q, k) [n,
    heads, head_dim], in new tensors or in ``out``, which may be (q, k)."""
    D, turns = plan.head_dim, plan.turns
    some = q if q is not None else k
    if some is None:
        raise ValueError("rope: neither queries nor keys")
    dt = some.dtype
    if dt not in _KV_ROWS:
        raise ValueError(f"rope: rows are {dt}, not one of {[str(d) for d in _KV_ROWS]}")
    n, Hq, qs = _rope_rows("q", q, D, dt)
    k_rows, Hk, ks = _rope_rows("k", k, D, dt)
    if q is None:
        n = k_rows
    elif k is not None and k_rows != n:
        raise ValueError(f"rope: {n} rows of q and {k_rows} of k")
    _packed("rope", "positions", positions, torch.int32, (n,))
    for name, t, w in (("q", q, q_weight), ("k", k, k_weight)):
        if w is not None:
            if t is None:
                raise ValueError(f"rope: a weight of {name} without {name}")
            _packed("rope", f"the weight of {name}", w, dt, (D,))
    if out is None:
        q_out = None if q is None else q.new_empty((n, Hq, D))
        k_out = None if k is None else k.new_empty((n, Hk, D))
        out, qos, kos = (q_out, k_out), Hq * D, Hk * D
    else:
        q_out, k_out = out
        if (q_out is None) != (q is None) or (k_out is None) != (k is None):
            raise ValueError("rope: results for the sides that are given, and for no others")
        qo_rows, qo_heads, qos = _rope_rows("the result of q", q_out, D, dt)
        ko_rows, ko_heads, kos = _rope_rows("the result of k", k_out, D, dt)
        if (q is not None and (qo_rows, qo_heads) != (n, Hq)) or (k is not None and (ko_rows, ko_heads) != (n, Hk)):
            raise ValueError(f"rope: results of {qo_rows} x {qo_heads} and {ko_rows} x {ko_heads} heads for "
                             f"{n} x {Hq} and {n} x {Hk}")
    _on_one_gpu("rope", positions, q, k, turns, q_weight, k_weight, q_out, k_out)
    lib().call("lhq_rope_f32" if dt == torch.float32 else "lhq_rope_bf16", P(q), qs, P(k), ks, positions.data_ptr(),
               turns.data_ptr(), P(q_weight), P(k_weight), eps, plan.gain, P(q_out), qos, P(k_out), kos,
               int(plan.interleaved), n, Hq, Hk, D, plan.rot_dim, stream())
    return out


def _rope_rows(name: str, t: torch.Tensor | None, D: int, dt) -> tuple[int, int, int]:
    """(rows, heads, the stride between rows) of one side, zeros where there is none."""
    if t is None:
        return 0, 0, 0
    shape = t.shape
    heads = shape[1] // D if len(shape) == 2 else shape[1] if len(shape) == 3 else 0
    n, stride = _kv_rows("rope", name, t, heads, D, (dt,))
    return n, heads, stride


def prefill_workspace(n_seqs: int, n: int, n_heads: int, n_kv_heads: int, head_dim: int) -> torch.Tensor | None:
    """A device workspace of the size that attn_prompt and kv_prefill can use (None: they need none)."""
    nbytes = lib().lhq_prefill_workspace_bytes(n_seqs, n, n_heads, n_kv_heads, head_dim)
    return empty((nbytes,), np.uint8) if nbytes > 0 else None


def _prefill_rows(fn: str, q: torch.Tensor, k: torch.Tensor | None, v: torch.Tensor | None, H: int | None, D: int,
                  out: torch.Tensor | None, workspace: torch.Tensor | None):
    """Checks rows, result and workspace; returns (n, heads, kv heads, strides, out, whether it was made here, workspace bytes)."""
    shape = q.shape
    heads = shape[1] // D if len(shape) == 2 else shape[1] if len(shape) == 3 else 0
    n, qs = _kv_rows(fn, "q", q, heads, D, _KV_BITS)
    if (k is None) != (v is None):
        raise ValueError(f"{fn}: new keys without values, or values without keys")
    ks = vs = 0
    if k is not None:
        if H is None:
            H = k.shape[1] // D if k.dim() == 2 else k.shape[1] if k.dim() == 3 else 0
        n_keys, ks = _kv_rows(fn, "k", k, H, D, _KV_BITS)
        n_values, vs = _kv_rows(fn, "v", v, H, D, _KV_BITS)
        if n_keys != n or n_values != n:
            raise ValueError(f"{fn}: {n} queries with {n_keys} new keys and {n_values} values")
    if not H or heads == 0 or heads % H != 0:
        raise ValueError(f"{fn}: {heads} query heads over {H} kv heads")
    made = out is None
    if made:
        out = q.new_empty((n, heads, D))
    elif out.dtype != torch.int16 or out.numel() != n * heads * D or not out.is_contiguous():
        raise ValueError(f"{fn}: out must be contiguous [{n}, {heads}, {D}] int16")
    nbytes = 0
    if workspace is not None:
        if not workspace.is_contiguous():
            raise ValueError(f"{fn}: workspace must be contiguous (strides {tuple(workspace.stride())})")
        nbytes = workspace.numel() * workspace.element_size()
    return n, heads, H, (qs, ks, vs), out, int(made), nbytes


def attn_prompt(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, offsets: torch.Tensor, head_dim: int,
                scale: float | None = None, workspace: torch.Tensor | None = None,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of whole prompts, packed: q [n, heads * head_dim], k and v
    [n, kv heads * head_dim] (bf16 as int16 bits, rows may be strided), sequence s
    having rows offsets[s] .. offsets[s + 1] (int32 [B + 1]).  Returns out [n,
    heads, head_dim], int16 bits; rows that offsets give to no sequence are not
    computed: zeros in a result that is made here, else what ``out`` held.  ``out``
    may be q itself where its rows lie one after the other, and else overlaps none of
    q, k and v."""
    fn, D = "attn_prompt", head_dim
    if D < 1:
        raise ValueError(f"{fn}: head_dim {D}")
    if offsets.dtype is not torch.int32 or offsets.dim() != 1 or offsets.shape[0] == 0 or not offsets.is_contiguous():
        raise ValueError(f"{fn}: offsets must be contiguous [B + 1] int32, got {tuple(offsets.shape)} {offsets.dtype}")
    n, heads, H, (qs, ks, vs), out, made, nbytes = _prefill_rows(fn, q, k, v, None, D, out, workspace)
    _on_one_gpu(fn, q, k, v, offsets, workspace, out)
    lib().call("lhq_attn_prompt_bf16", q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, offsets.data_ptr(),
               out.data_ptr(), offsets.shape[0] - 1, n, heads, H, D, D ** -0.5 if scale is None else scale,
               made, P(workspace), nbytes, stream())
    return out


def kv_prefill(cache: KvCache, q: torch.Tensor, offsets: torch.Tensor, lengths: torch.Tensor,
               block_table: torch.Tensor, k_new: torch.Tensor | None, v_new: torch.Tensor | None,
               scale: float | None = None, workspace: torch.Tensor | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of any number of new tokens a sequence over its first lengths[s]
    cached tokens and, causal, over the new ones: kv_attn without its bound of 64
    and without trees.  Rows as in attn_prompt.  Returns out [n, heads, head_dim],
    int16 bits; rows that offsets give to no sequence are not computed: zeros in a
    result that is made here, else what ``out`` held."""
    fn, H, D = "kv_prefill", cache.n_kv_heads, cache.head_dim
    B, width = _kv_tables(fn, offsets, lengths, block_table)
    n, heads, H, (qs, ks, vs), out, made, nbytes = _prefill_rows(fn, q, k_new, v_new, H, D, out, workspace)
    _on_one_gpu(fn, cache.k, q, offsets, lengths, block_table, k_new, v_new, workspace, out)
    lib().call("lhq_kv_prefill_bf16", q.data_ptr(), qs, P(k_new), ks, P(v_new), vs, offsets.data_ptr(),
               lengths.data_ptr(), block_table.data_ptr(), *cache.pointers(), out.data_ptr(), _KV_FORMATS[cache.fmt],
               B, n, width, cache.n_pages, heads, H, D, D ** -0.5 if scale is None else scale, made, P(workspace), nbytes,
               stream())
    return out
