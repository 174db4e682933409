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

The arithmetic lives in ``libecah_sampler.so``; its torch binding
(csrc/binding.cpp) checks tensors and launches on the current torch stream.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _abi
from ._abi import binding, lib
from .sampler import _LIB, resolve_device

_DTYPES = {torch.float16: _abi.DTYPE_F16, torch.bfloat16: _abi.DTYPE_BF16}
E4M3 = torch.float8_e4m3fn
HEAD_DIMS = (64, 96, 128, 192, 256)


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
    return binding().append(q, k, v, positions, batch_index, kv_indptr, kv_indices, k_cache, v_cache, k_scale, v_scale,
                            cos_sin, q_norm, k_norm, eps, interleaved, q_out, None)


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
    tokens).  ``workspace``: zero-filled uint8, 16-byte aligned,
    one per concurrent stream."""
    got = binding().decode(q, kv_indptr, kv_indices, kv_last_page_len, k_cache, v_cache, workspace, k_scale, v_scale,
                           sm_scale, out, lse, None)
    return got if lse is None else got[0]


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
        self._layout = (num_qo_heads, num_kv_heads, head_dim, page_size, int(kv_dtype == E4M3), max_batch,
                        _DTYPES[dtype])
        self._append, self._decode = binding().append, binding().decode

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

    def append(self, q, k, v, positions, batch_index, kv_indptr, kv_indices, k_cache, v_cache, *, k_scale=None,
               v_scale=None, cos_sin=None, q_norm=None, k_norm=None, eps=1e-6, interleaved=False, q_out=None):
        """``append`` with this model's layout checked."""
        return self._append(q, k, v, positions, batch_index, kv_indptr, kv_indices, k_cache, v_cache, k_scale,
                            v_scale, cos_sin, q_norm, k_norm, eps, interleaved, q_out, self._layout)

    def decode(self, q, kv_indptr, kv_indices, kv_last_page_len, k_cache, v_cache, *, k_scale=None, v_scale=None,
               sm_scale=None, out=None, lse=None, return_lse: bool = False):
        """``decode`` with this model's layout checked and its workspace;
        ``(out, lse)`` with ``return_lse``."""
        if lse is None and return_lse:
            lse = True
        got = self._decode(q, kv_indptr, kv_indices, kv_last_page_len, k_cache, v_cache, self.workspace, k_scale,
                           v_scale, sm_scale, out, lse, self._layout)
        return got[0] if lse is not None and not return_lse else got


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
    if q is not None and q_out is None:
        raise RuntimeError("q_out is required with q")
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
