"""The paged key-value cache: ``PagedAttention`` (and the functions ``append``,
``decode``, ``prefill`` and ``copy_pages`` it calls, and the torch custom ops
``torch.ops.ecah.paged_append`` / ``paged_decode`` / ``paged_prefill`` /
``paged_copy``).

``append`` normalises and rotates the new tokens' queries and keys and writes
keys and values into their cache pages -- as they are, or as 8-bit floats with
a scale per token and head; ``decode`` attends one new token per request over
the pages, ``prefill`` several (a prompt, a chunk of one, drafted tokens);
``copy_pages`` copies pages in all layers, to fork requests.  Pages are listed per request as the reference lists them for its
attention (``kv_indptr`` / ``kv_indices`` / ``kv_last_page_len``,
ecahlang/manager.py:228-253), so its page allocator feeds all calls
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


def prefill_workspace_bytes(head_dim: int) -> int:
    """Workspace of any ``prefill`` launch with heads of `head_dim` on the
    current device."""
    return int(lib().ecah_paged_prefill_workspace_bytes(head_dim))


def prefill(q: torch.Tensor, qo_indptr: torch.Tensor, kv_indptr: torch.Tensor, kv_indices: torch.Tensor,
            kv_last_page_len: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, workspace: torch.Tensor, *,
            k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None, causal: bool = True,
            sm_scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
            lse: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Enqueue the attention of ``q`` [T, Hq, D], the requests' new tokens one
    request behind another, over the requests' cached keys and values (the new
    tokens' own among them: ``append`` comes first); returns ``out`` [T, Hq, D]
    (allocated unless given).

    Request b's tokens are ``q[qo_indptr[b]:qo_indptr[b + 1]]`` (``qo_indptr``
    int32 [batch + 1], not decreasing), the last of its cached ones; token i of
    n sees the first ``len - n + i + 1`` keys if ``causal``, else all ``len``.
    A token that sees no key gets zeros.  Rows outside every request (padding
    behind the last one) are neither read nor written.  ``lse`` float32
    [T, Hq], ``sm_scale``, the page lists and the cache as ``decode`` takes
    them.  ``workspace``: zero-filled uint8, 16-byte aligned, one per
    concurrent stream."""
    got = binding().prefill(q, qo_indptr, kv_indptr, kv_indices, kv_last_page_len, k_cache, v_cache, workspace, k_scale,
                            v_scale, causal, sm_scale, out, lse, None)
    return got if lse is None else got[0]


def _pages(src, dst, tokens, num_pages: int, page_size: int, device):
    """``copy_pages``'s lists as device tensors; host sequences are checked first."""
    on_device = [torch.is_tensor(t) and t.is_cuda for t in (src, dst)]
    if all(on_device):
        return src, dst, tokens
    if any(on_device) or (torch.is_tensor(tokens) and tokens.is_cuda):
        raise RuntimeError("src, dst and tokens must all be device tensors, or all host sequences")
    src, dst = ([int(p) for p in t] for t in (src, dst))
    if len(src) != len(dst):
        raise RuntimeError(f"{len(src)} source and {len(dst)} destination pages")
    if any(not 0 <= p < num_pages for p in src + dst):
        raise IndexError(f"page outside [0, {num_pages})")
    if len(set(dst)) != len(dst) or set(dst) & set(src):
        raise RuntimeError("destination pages must differ from each other and from every source")
    if tokens is not None:
        tokens = [int(n) for n in tokens]
        if len(tokens) != len(src) or any(not 0 <= n <= page_size for n in tokens):
            raise RuntimeError(f"tokens must be {len(src)} numbers in [0, {page_size}]")
        tokens = torch.tensor(tokens, dtype=torch.int32).to(device, non_blocking=True)
    return (*(torch.tensor(t, dtype=torch.int32).to(device, non_blocking=True) for t in (src, dst)), tokens)


def _copy(caches, src, dst, tokens, layout) -> None:
    caches = list(caches)
    if not caches:
        return
    k = caches[0][0]
    if not torch.is_tensor(k) or k.dim() != 4:
        raise RuntimeError("caches must be (k_cache, v_cache, k_scale, v_scale) of each layer")
    src, dst, tokens = _pages(src, dst, tokens, k.shape[0], k.shape[1], k.device)
    binding().copy_pages(src, dst, tokens, caches, layout)


def copy_pages(src, dst, caches, *, tokens=None) -> None:
    """Enqueue the copy of pages ``src[i]`` to ``dst[i]`` in every layer of
    ``caches``, a sequence of ``(k_cache, v_cache, k_scale, v_scale)`` of one
    shape (as ``PagedAttention.new_cache`` gives them); one launch for up to 64
    layers.

    ``tokens``: copy the first ``tokens[i]`` slots of the page alone (None:
    all).  To fork a request, list its whole pages in the child's page list and
    copy its last page, ``kv_last_page_len`` tokens of it.  Destinations must
    differ from each other and from every source.  ``src``, ``dst`` and
    ``tokens`` are int32 tensors on the device, used as they are (pairs with a
    page outside the cache, such as -1, are skipped; for captured calls), or
    host sequences, which are checked and copied to it."""
    _copy(caches, src, dst, tokens, None)


class PagedAttention:
    """One model's paged attention on one stream: its head layout and the
    workspaces, shared by all layers (``prefill``'s is made by its first call,
    which has to be outside a capture).

    ``kv_dtype`` is the model dtype (default) or ``torch.float8_e4m3fn``;
    ``max_batch`` bounds the requests of one ``decode`` or ``prefill``."""

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
        self._prefill_workspace: Optional[torch.Tensor] = None
        self._layout = (num_qo_heads, num_kv_heads, head_dim, page_size, int(kv_dtype == E4M3), max_batch,
                        _DTYPES[dtype])
        self._append, self._decode, self._prefill = binding().append, binding().decode, binding().prefill

    @property
    def prefill_workspace(self) -> torch.Tensor:
        """``prefill``'s workspace (39 MB), made by the first ``prefill``, so that
        a handle that only decodes holds none.  Not inside a CUDA-graph capture,
        where it would be zero-filled by that graph's replays alone."""
        if self._prefill_workspace is None:
            if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("the workspace of prefill cannot be made inside a CUDA-graph capture: "
                                   "call prefill once before it, or read prefill_workspace")
            with torch.cuda.device(self.device):
                n = prefill_workspace_bytes(self.head_dim)
            self._prefill_workspace = torch.zeros(n, dtype=torch.uint8, device=self.device)
        return self._prefill_workspace

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

    def prefill(self, q, qo_indptr, kv_indptr, kv_indices, kv_last_page_len, k_cache, v_cache, *, k_scale=None,
                v_scale=None, causal: bool = True, sm_scale=None, out=None, lse=None, return_lse: bool = False):
        """``prefill`` with this model's layout checked and its workspace;
        ``(out, lse)`` with ``return_lse``."""
        if lse is None and return_lse:
            lse = True
        got = self._prefill(q, qo_indptr, kv_indptr, kv_indices, kv_last_page_len, k_cache, v_cache,
                            self._prefill_workspace if self._prefill_workspace is not None else self.prefill_workspace, k_scale, v_scale, causal, sm_scale, out, lse, self._layout)
        return got[0] if lse is not None and not return_lse else got

    def copy_pages(self, src, dst, caches, *, tokens=None) -> None:
        """``copy_pages`` with this model's layout checked."""
        _copy(caches, src, dst, tokens, self._layout)


# ----------------------------------------------------------- torch custom ops
_LIB.define(
    "paged_append(Tensor? q, Tensor k, Tensor v, Tensor positions, Tensor batch_index, Tensor kv_indptr, "
    "Tensor kv_indices, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!)? k_scale, Tensor(d!)? v_scale, "
    "Tensor? cos_sin, Tensor? q_norm, Tensor? k_norm, float eps, bool interleaved, Tensor(e!)? q_out) -> ()")
_LIB.define(
    "paged_decode(Tensor q, Tensor kv_indptr, Tensor kv_indices, Tensor kv_last_page_len, Tensor k_cache, "
    "Tensor v_cache, Tensor? k_scale, Tensor? v_scale, float sm_scale, Tensor(a!) out, Tensor(b!)? lse, "
    "Tensor(c!) workspace) -> ()")
_LIB.define(
    "paged_prefill(Tensor q, Tensor qo_indptr, Tensor kv_indptr, Tensor kv_indices, Tensor kv_last_page_len, "
    "Tensor k_cache, Tensor v_cache, Tensor? k_scale, Tensor? v_scale, bool causal, float sm_scale, Tensor(a!) out, "
    "Tensor(b!)? lse, Tensor(c!) workspace) -> ()")
_LIB.define(
    "paged_copy(Tensor src, Tensor dst, Tensor? tokens, Tensor(a!)[] k_caches, Tensor(b!)[] v_caches, "
    "Tensor(c!)[] k_scales, Tensor(d!)[] v_scales) -> ()")


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


def _prefill_op_cuda(q, qo_indptr, kv_indptr, kv_indices, kv_last_page_len, k_cache, v_cache, k_scale, v_scale, causal,
                     sm_scale, out, lse, workspace):
    prefill(q, qo_indptr, kv_indptr, kv_indices, kv_last_page_len, k_cache, v_cache, workspace, k_scale=k_scale,
            v_scale=v_scale, causal=causal, sm_scale=sm_scale, out=out, lse=lse)


def _copy_op_cuda(src, dst, tokens, k_caches, v_caches, k_scales, v_scales):
    """Empty lists of scales for caches in the model dtype."""
    none = [None] * len(k_caches)
    for name, t in (("v_caches", v_caches), ("k_scales", k_scales or none), ("v_scales", v_scales or none)):
        if len(t) != len(k_caches):
            raise RuntimeError(f"{name}: expected {len(k_caches)} layers, got {len(t)}")
    copy_pages(src, dst, list(zip(k_caches, v_caches, k_scales or none, v_scales or none)), tokens=tokens)


_LIB.impl("paged_append", _append_op_cuda, "CUDA")
_LIB.impl("paged_decode", _decode_op_cuda, "CUDA")
_LIB.impl("paged_prefill", _prefill_op_cuda, "CUDA")
_LIB.impl("paged_copy", _copy_op_cuda, "CUDA")


@torch.library.register_fake("ecah::paged_append")
def _append_op_fake(q, k, v, positions, batch_index, kv_indptr, kv_indices, k_cache, v_cache, k_scale, v_scale,
                    cos_sin, q_norm, k_norm, eps, interleaved, q_out):
    return None


@torch.library.register_fake("ecah::paged_decode")
def _decode_op_fake(q, kv_indptr, kv_indices, kv_last_page_len, k_cache, v_cache, k_scale, v_scale, sm_scale, out,
                    lse, workspace):
    return None


@torch.library.register_fake("ecah::paged_prefill")
def _prefill_op_fake(q, qo_indptr, kv_indptr, kv_indices, kv_last_page_len, k_cache, v_cache, k_scale, v_scale, causal,
                     sm_scale, out, lse, workspace):
    return None


@torch.library.register_fake("ecah::paged_copy")
def _copy_op_fake(src, dst, tokens, k_caches, v_caches, k_scales, v_scales):
    return None
