"""The decode step's paged key-value cache: ``PagedAttention`` (and the
functions ``append`` and ``decode`` it calls, and the torch custom ops
``torch.ops.ecah.paged_append`` / ``paged_decode``).

``append`` normalises and rotates the new tokens' queries and keys and writes
keys and values into their cache pages -- as they are, or as 8-bit floats with
a scale per token and head; ``decode`` attends one new token per request over
the pages.  Pages are listed per request as the reference lists them for its
attention (``kv_indptr`` / ``kv_indices`` / ``kv_last_page_len``,
ecahlang/manager.py:228-253), so its page allocator feeds both calls
(manager.py:143-185 and main.py:68 are the calls they replace).

The arithmetic lives in ``libecah_sampler.so``; this module checks tensors and
launches on the current torch stream.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import _abi
from ._abi import AppendArgs, DecodeArgs, check, lib
from .sampler import _LIB, _need, on_device, resolve_device

_DTYPES = {torch.float16: _abi.DTYPE_F16, torch.bfloat16: _abi.DTYPE_BF16}
E4M3 = torch.float8_e4m3fn
HEAD_DIMS = (64, 96, 128, 192, 256)


def _rows(t: torch.Tensor, name: str, shape, dtype, dev) -> Tuple[int, int]:
    """Token and head strides of a [tokens, heads, head_dim] tensor."""
    if t.dtype != dtype or t.device != dev:
        raise RuntimeError(f"{name}: expected {dtype} on {dev}, got {t.dtype} on {t.device}")
    if t.shape != shape:
        raise RuntimeError(f"{name}: expected shape {list(shape)}, got {list(t.shape)}")
    st, sh, sd = t.stride()
    if shape[0] <= 1:
        st = 0
    if shape[1] <= 1:
        sh = 0
    if sd != 1 or st % 8 or sh % 8 or t.data_ptr() % 16:
        raise RuntimeError(f"{name}: rows of head_dim must be contiguous and 16-byte aligned")
    return st, sh


def _fill_cache(c, dtype, dev, k_cache, v_cache, k_scale, v_scale, kv_indptr, kv_indices) -> None:
    """Checks the cache tensors and fills struct ecah_kv_cache."""
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape:
        raise RuntimeError("k_cache and v_cache must be [num_pages, page_size, num_kv_heads, head_dim]")
    kv = k_cache.dtype
    if kv != dtype and kv != E4M3 or v_cache.dtype != kv:
        raise RuntimeError(f"cache must be {dtype} or {E4M3}, got {kv} and {v_cache.dtype}")
    if k_cache.device != dev or v_cache.device != dev:
        raise RuntimeError(f"cache must be on {dev}")
    pages, page, heads, D = k_cache.shape
    if D not in HEAD_DIMS:
        raise RuntimeError(f"head_dim {D} is not one of {HEAD_DIMS}")
    if page < 1 or heads < 1:
        raise RuntimeError("page_size and num_kv_heads must be positive")
    unit = 16 if kv == E4M3 else 8
    got = []
    for t, name in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        sp, ss, sh, sd = t.stride()
        if pages <= 1:
            sp = 0
        if page == 1:
            ss = 0
        if heads == 1:
            sh = 0
        if sd != 1 or sp % unit or ss % unit or sh % unit or t.data_ptr() % 16:
            raise RuntimeError(f"{name}: rows of head_dim must be contiguous and 16-byte aligned")
        got += [sp, ss, sh]
    c.k_page_stride, c.k_slot_stride, c.k_head_stride, c.v_page_stride, c.v_slot_stride, c.v_head_stride = got
    if kv == E4M3:
        if k_scale is None or v_scale is None:
            raise RuntimeError("an e4m3 cache needs k_scale and v_scale")
        for t, name in ((k_scale, "k_scale"), (v_scale, "v_scale")):
            if t.shape != (pages, heads, page):
                raise RuntimeError(f"{name}: expected shape [num_pages, num_kv_heads, page_size]")
            _need(t, name, torch.float32, pages * heads * page, dev)
        c.kv_dtype, c.k_scale, c.v_scale = _abi.KV_E4M3, k_scale.data_ptr(), v_scale.data_ptr()
    else:
        if k_scale is not None or v_scale is not None:
            raise RuntimeError(f"a {kv} cache takes no scales")
        c.kv_dtype = _DTYPES[kv]
    n = kv_indptr.numel()
    if n < 1:
        raise RuntimeError("kv_indptr must have batch + 1 entries")
    _need(kv_indptr, "kv_indptr", torch.int32, n, dev)
    _need(kv_indices, "kv_indices", torch.int32, kv_indices.numel(), dev)
    c.num_pages, c.page_size, c.num_kv_heads, c.head_dim, c.batch = pages, page, heads, D, n - 1
    c.k_cache, c.v_cache = k_cache.data_ptr(), v_cache.data_ptr()
    c.kv_indptr, c.kv_indices, c.num_indices = kv_indptr.data_ptr(), kv_indices.data_ptr(), kv_indices.numel()


def append(q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
           batch_index: torch.Tensor, kv_indptr: torch.Tensor, kv_indices: torch.Tensor, k_cache: torch.Tensor,
           v_cache: torch.Tensor, *, k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None,
           cos_sin: Optional[torch.Tensor] = None, q_norm: Optional[torch.Tensor] = None,
           k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6, interleaved: bool = False,
           q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Enqueue one append of T tokens; returns the queries, normalised and
    rotated (``q_out``, allocated unless given; ``q`` itself is allowed).

    ``q`` [T, Hq, D] (or None), ``k`` and ``v`` [T, Hk, D]: views into a packed
    projection are fine.  ``positions`` int32 [T] give both the rotation's row
    of ``cos_sin`` (float32 [rows, D]: cosines then sines; None: no rotation)
    and the cache slot, in the pages of request ``batch_index`` int32 [T] (-1:
    a padding row, nothing is written).  ``q_norm`` / ``k_norm`` [D]: weights
    of the per-head RMS norm (None: no norm).  ``interleaved`` pairs (2i, 2i+1)
    instead of (i, i + D/2).  For a ``torch.float8_e4m3fn`` cache the scales go
    to ``k_scale`` / ``v_scale`` float32 [num_pages, Hk, page_size]."""
    dt = _DTYPES.get(k.dtype)
    if dt is None:
        raise RuntimeError(f"unsupported dtype {k.dtype}: append takes float16 and bfloat16")
    if not k.is_cuda:
        raise RuntimeError("append needs CUDA tensors (there is no CPU path)")
    dev = k.device
    a = AppendArgs()
    _fill_cache(a.cache, k.dtype, dev, k_cache, v_cache, k_scale, v_scale, kv_indptr, kv_indices)
    heads, D = a.cache.num_kv_heads, a.cache.head_dim
    T = k.shape[0]
    a.k_token_stride, a.k_head_stride = _rows(k, "k", (T, heads, D), k.dtype, dev)
    a.v_token_stride, a.v_head_stride = _rows(v, "v", (T, heads, D), k.dtype, dev)
    if q is not None:
        if q.dim() != 3 or q.shape[1] < 1:
            raise RuntimeError("q must be [T, num_qo_heads, head_dim]")
        shape = (T, q.shape[1], D)
        a.q_token_stride, a.q_head_stride = _rows(q, "q", shape, k.dtype, dev)
        if q_out is None:
            q_out = torch.empty(shape, dtype=k.dtype, device=dev)
        a.qo_token_stride, a.qo_head_stride = _rows(q_out, "q_out", shape, k.dtype, dev)
        a.q, a.q_out, a.num_qo_heads = q.data_ptr(), q_out.data_ptr(), shape[1]
    elif q_out is not None or q_norm is not None:
        raise RuntimeError("q_out and q_norm need q")
    _need(positions, "positions", torch.int32, T, dev)
    _need(batch_index, "batch_index", torch.int32, T, dev)
    if q_norm is not None:
        _need(q_norm, "q_norm", k.dtype, D, dev)
        a.q_norm = q_norm.data_ptr()
    if k_norm is not None:
        _need(k_norm, "k_norm", k.dtype, D, dev)
        a.k_norm = k_norm.data_ptr()
    if cos_sin is not None:
        if cos_sin.dim() != 2 or cos_sin.shape[0] < 1 or cos_sin.shape[1] != D:
            raise RuntimeError(f"cos_sin must be [rows, {D}], got {list(cos_sin.shape)}")
        _need(cos_sin, "cos_sin", torch.float32, cos_sin.numel(), dev)
        a.cos_sin, a.table_rows = cos_sin.data_ptr(), cos_sin.shape[0]
    a.abi_version, a.dtype, a.tokens = _abi.ABI_VERSION, dt, T
    a.k, a.v, a.positions, a.batch_index = k.data_ptr(), v.data_ptr(), positions.data_ptr(), batch_index.data_ptr()
    a.eps, a.interleaved = eps, interleaved
    st = on_device(dev, lib().ecah_paged_append, a)
    if st:
        check(st, "ecah_paged_append")
    return q_out


def decode_workspace_bytes(batch: int, num_qo_heads: int, num_kv_heads: int, head_dim: int) -> int:
    """Workspace of ``decode`` launches of up to `batch` requests on the
    current device."""
    return int(lib().ecah_paged_decode_workspace_bytes(batch, num_qo_heads, num_kv_heads, head_dim))


def decode(q: torch.Tensor, kv_indptr: torch.Tensor, kv_indices: torch.Tensor, kv_last_page_len: torch.Tensor,
           k_cache: torch.Tensor, v_cache: torch.Tensor, workspace: torch.Tensor, *,
           k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None,
           sm_scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
           lse: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Enqueue the attention of ``q`` [batch, Hq, D], one new token per request,
    over the requests' cached keys and values; returns ``out`` [batch, Hq, D]
    (allocated unless given).

    Request b has ``(pages - 1) * page_size + kv_last_page_len[b]`` tokens; one
    without pages gets zeros.  ``sm_scale`` defaults to ``1 / sqrt(D)``.
    ``lse`` float32 [batch, Hq], when given, receives the natural logarithm of
    the softmax denominators (to join partial attentions; -inf without
    tokens).  ``workspace``: zero-filled uint8, one per concurrent stream."""
    dt = _DTYPES.get(q.dtype)
    if dt is None:
        raise RuntimeError(f"unsupported dtype {q.dtype}: decode takes float16 and bfloat16")
    if not q.is_cuda:
        raise RuntimeError("decode needs CUDA tensors (there is no CPU path)")
    dev = q.device
    a = DecodeArgs()
    c = a.cache
    _fill_cache(c, q.dtype, dev, k_cache, v_cache, k_scale, v_scale, kv_indptr, kv_indices)
    heads, D, B = c.num_kv_heads, c.head_dim, c.batch
    if q.dim() != 3 or q.shape[1] < 1 or q.shape[1] % heads:
        raise RuntimeError(f"q must be [{B}, num_qo_heads, {D}] with num_qo_heads a multiple of {heads}")
    Hq = q.shape[1]
    shape = (B, Hq, D)
    a.q_token_stride, a.q_head_stride = _rows(q, "q", shape, q.dtype, dev)
    if out is None:
        out = torch.empty(shape, dtype=q.dtype, device=dev)
    a.out_token_stride, a.out_head_stride = _rows(out, "out", shape, q.dtype, dev)
    if lse is not None:
        _need(lse, "lse", torch.float32, B * Hq, dev)
        a.lse = lse.data_ptr()
    _need(kv_last_page_len, "kv_last_page_len", torch.int32, B, dev)
    if workspace.device != dev or workspace.dtype != torch.uint8 or not workspace.is_contiguous():
        raise RuntimeError("workspace must be a contiguous uint8 tensor on q's device")
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(D)
    elif not (0.0 < sm_scale < math.inf):
        raise RuntimeError(f"sm_scale must be positive and finite, got {sm_scale}")
    a.abi_version, a.dtype, a.num_qo_heads, a.sm_scale = _abi.ABI_VERSION, dt, Hq, sm_scale
    a.q, a.out, a.kv_last_page_len = q.data_ptr(), out.data_ptr(), kv_last_page_len.data_ptr()
    a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.numel()
    st = on_device(dev, lib().ecah_paged_decode, a)
    if st:
        check(st, "ecah_paged_decode")
    return out


class PagedAttention:
    """One model's paged attention on one stream: its head layout and the
    decode workspace, shared by all layers.

    ``kv_dtype`` is the model dtype (default) or ``torch.float8_e4m3fn``;
    ``max_batch`` bounds the requests of one ``decode``."""

    def __init__(self, num_qo_heads: int, num_kv_heads: int, head_dim: int, page_size: int, dtype: torch.dtype,
                 kv_dtype: Optional[torch.dtype] = None, max_batch: int = 128, device="cuda"):
        if dtype not in _DTYPES:
            raise RuntimeError(f"unsupported model dtype {dtype}")
        kv_dtype = dtype if kv_dtype is None else kv_dtype
        if kv_dtype not in (dtype, E4M3):
            raise RuntimeError(f"kv_dtype must be {dtype} or {E4M3}, got {kv_dtype}")
        if head_dim not in HEAD_DIMS:
            raise RuntimeError(f"head_dim {head_dim} is not one of {HEAD_DIMS}")
        if num_kv_heads < 1 or num_qo_heads < 1 or num_qo_heads % num_kv_heads:
            raise RuntimeError("num_qo_heads must be a multiple of num_kv_heads")
        if page_size < 1 or max_batch < 1:
            raise RuntimeError("page_size and max_batch must be positive")
        self.num_qo_heads, self.num_kv_heads, self.head_dim = num_qo_heads, num_kv_heads, head_dim
        self.page_size, self.dtype, self.kv_dtype, self.max_batch = page_size, dtype, kv_dtype, max_batch
        self.device = resolve_device(device)
        with torch.cuda.device(self.device):
            n = decode_workspace_bytes(max_batch, num_qo_heads, num_kv_heads, head_dim)
        self.workspace = torch.zeros(n, dtype=torch.uint8, device=self.device)

    def new_cache(self, num_pages: int):
        """(k_cache, v_cache, k_scale, v_scale) of one layer, zero-filled; the
        scales are None for a cache in the model dtype."""
        shape = (num_pages, self.page_size, self.num_kv_heads, self.head_dim)
        e4m3 = self.kv_dtype == E4M3
        raw = torch.uint8 if e4m3 else self.dtype
        k, v = (torch.zeros(shape, dtype=raw, device=self.device).view(self.kv_dtype) for _ in range(2))
        if not e4m3:
            return k, v, None, None
        s = (num_pages, self.num_kv_heads, self.page_size)
        return k, v, torch.zeros(s, device=self.device), torch.zeros(s, device=self.device)

    def _check(self, k_cache, q):
        if k_cache.dtype != self.kv_dtype or k_cache.shape[1:] != (self.page_size, self.num_kv_heads, self.head_dim):
            raise RuntimeError(f"cache must be [pages, {self.page_size}, {self.num_kv_heads}, {self.head_dim}] "
                               f"{self.kv_dtype}, got {list(k_cache.shape)} {k_cache.dtype}")
        if q is not None and (q.dtype != self.dtype or q.dim() != 3 or q.shape[1] != self.num_qo_heads):
            raise RuntimeError(f"q must be [tokens, {self.num_qo_heads}, {self.head_dim}] {self.dtype}, "
                               f"got {list(q.shape)} {q.dtype}")

    def append(self, q, k, v, positions, batch_index, kv_indptr, kv_indices, k_cache, v_cache, **kw):
        """``append`` with this model's layout checked."""
        self._check(k_cache, q)
        return append(q, k, v, positions, batch_index, kv_indptr, kv_indices, k_cache, v_cache, **kw)

    def decode(self, q, kv_indptr, kv_indices, kv_last_page_len, k_cache, v_cache, *, return_lse: bool = False, **kw):
        """``decode`` with this model's layout checked and its workspace;
        ``(out, lse)`` with ``return_lse``."""
        self._check(k_cache, q)
        if q.shape[0] > self.max_batch:
            raise RuntimeError(f"{q.shape[0]} requests, max_batch is {self.max_batch}")
        if return_lse:
            lse = kw.pop("lse", None)
            if lse is None:
                lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
            return decode(q, kv_indptr, kv_indices, kv_last_page_len, k_cache, v_cache, self.workspace, lse=lse,
                          **kw), lse
        return decode(q, kv_indptr, kv_indices, kv_last_page_len, k_cache, v_cache, self.workspace, **kw)


# ----------------------------------------------------------- torch custom ops
_LIB.define(
    "paged_append(Tensor? q, Tensor k, Tensor v, Tensor positions, Tensor batch_index, Tensor kv_indptr, "
    "Tensor kv_indices, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!)? k_scale, Tensor(d!)? v_scale, "
    "Tensor? cos_sin, Tensor? q_norm, Tensor? k_norm, float eps, bool interleaved, Tensor(e!)? q_out) -> ()")
_LIB.define(
    "paged_decode(Tensor q, Tensor kv_indptr, Tensor kv_indices, Tensor kv_last_page_len, Tensor k_cache, "
    "Tensor v_cache, Tensor? k_scale, Tensor? v_scale, float sm_scale, Tensor(a!) out, Tensor(b!)? lse, "
    "Tensor(c!) workspace) -> ()")


def _append_op_cuda(q, k, v, positions, batch_index, kv_indptr, kv_indices, k_cache, v_cache, k_scale, v_scale,
                    cos_sin, q_norm, k_norm, eps, interleaved, q_out):
    append(q, k, v, positions, batch_index, kv_indptr, kv_indices, k_cache, v_cache, k_scale=k_scale,
           v_scale=v_scale, cos_sin=cos_sin, q_norm=q_norm, k_norm=k_norm, eps=eps, interleaved=interleaved,
           q_out=q_out)


def _decode_op_cuda(q, kv_indptr, kv_indices, kv_last_page_len, k_cache, v_cache, k_scale, v_scale, sm_scale, out,
                    lse, workspace):
    decode(q, kv_indptr, kv_indices, kv_last_page_len, k_cache, v_cache, workspace, k_scale=k_scale,
           v_scale=v_scale, sm_scale=sm_scale, out=out, lse=lse)


_LIB.impl("paged_append", _append_op_cuda, "CUDA")
_LIB.impl("paged_decode", _decode_op_cuda, "CUDA")


@torch.library.register_fake("ecah::paged_append")
def _append_op_fake(q, k, v, positions, batch_index, kv_indptr, kv_indices, k_cache, v_cache, k_scale, v_scale,
                    cos_sin, q_norm, k_norm, eps, interleaved, q_out):
    return None


@torch.library.register_fake("ecah::paged_decode")
def _decode_op_fake(q, kv_indptr, kv_indices, kv_last_page_len, k_cache, v_cache, k_scale, v_scale, sm_scale, out,
                    lse, workspace):
    return None
