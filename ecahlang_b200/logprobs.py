"""Token log probabilities: ``TokenLogprobs`` / ``launch`` and the torch custom
op ``torch.ops.ecah.token_logprobs``.

For every row of logits: the log probability of given tokens, the entropy of
the row's distribution and its most likely alternatives, in one read of the
logits -- the ``logprobs`` / ``top_logprobs`` fields of a completion, which the
reference does not offer (ecahlang/main.py:377-379 keeps the drawn id alone).
Works on a decode batch (the sampled ids) and on a prompt (every position's
next token).  The arithmetic lives in ``libecah_sampler.so``; this module
checks tensors and launches on the current torch stream.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _abi
from ._abi import LogprobArgs, check, lib
from .sampler import _DTYPES, _LIB, _need, on_device, resolve_device

MAX_TOP_N = _abi.MAX_TOP_N


class RowLogprobs(NamedTuple):
    """One launch's results.  ``top_ids`` is -1 (and ``top_logprobs`` -inf)
    past a row's last entry with mass."""
    logprobs: torch.Tensor       # float32, the shape of token_ids
    entropy: torch.Tensor        # float32 [R], natural units
    top_ids: torch.Tensor        # int32 [R, top_n]
    top_logprobs: torch.Tensor   # float32 [R, top_n]


def new_workspace(device="cuda") -> torch.Tensor:
    """Zero-filled workspace of any launch on `device`; one per stream that
    may run a launch concurrently."""
    dev = resolve_device(device)
    with torch.cuda.device(dev):
        n = int(lib().ecah_token_logprobs_workspace_bytes())
    return torch.zeros(n, dtype=torch.uint8, device=dev)


def launch(logits: torch.Tensor, token_ids: Optional[torch.Tensor], workspace: torch.Tensor, *, top_n: int = 0,
           temperature: Optional[torch.Tensor] = None, row_index: Optional[torch.Tensor] = None,
           logprobs: Optional[torch.Tensor] = None, entropy: Optional[torch.Tensor] = None,
           top_ids: Optional[torch.Tensor] = None, top_logprobs: Optional[torch.Tensor] = None) -> RowLogprobs:
    """Enqueue one launch over ``logits`` [R, V] (rows contiguous, any row
    stride; f16, bf16 or f32).

    ``token_ids`` int32 [R] or [R, K]: the tokens to score (None: none).  A
    token outside [0, V) has NaN.  ``top_n`` (at most 32): alternatives by
    logit, ties to the lower id.  ``temperature`` float32 [R] (None: 1) is the
    sampler's; T <= 0 is the greedy distribution.  ``row_index`` int32 [R]
    gathers rows of a larger [L, V] buffer, as in ``sampler.launch``.  The
    output tensors are allocated unless given (contiguous, the shapes of
    ``RowLogprobs``)."""
    if logits.dim() != 2:
        raise RuntimeError("logits must be [R, V]")
    dt = _DTYPES.get(logits.dtype)
    if dt is None:
        raise RuntimeError(f"unsupported logits dtype {logits.dtype}")
    if not logits.is_cuda:
        raise RuntimeError("logits must be a CUDA tensor (there is no CPU path)")
    L, V = logits.shape
    row_stride, col_stride = logits.stride()
    if V < 1 or (col_stride != 1 and V > 1):
        raise RuntimeError("logits rows must be contiguous and not empty")
    if not 0 <= top_n <= MAX_TOP_N:
        raise RuntimeError(f"top_n must be in [0, {MAX_TOP_N}], got {top_n}")
    dev = logits.device
    a = LogprobArgs()
    R = L
    if row_index is not None:
        R = row_index.numel()
        _need(row_index, "row_index", torch.int32, R, dev)
        if L < 1 and R:
            raise RuntimeError("row_index into logits without rows")
        a.row_index, a.logit_rows = row_index.data_ptr(), L
    K = 0
    shape = (R, 0)
    if token_ids is not None:
        shape = token_ids.shape
        if len(shape) not in (1, 2) or shape[0] != R:
            raise RuntimeError(f"token_ids must be [{R}] or [{R}, K], got {list(shape)}")
        K = shape[1] if len(shape) == 2 else 1
        _need(token_ids, "token_ids", torch.int32, R * K, dev)
        a.token_ids = token_ids.data_ptr()
    if temperature is not None:
        _need(temperature, "temperature", torch.float32, R, dev)
        a.temperature = temperature.data_ptr()
    if workspace.device != dev or workspace.dtype != torch.uint8 or not workspace.is_contiguous():
        raise RuntimeError("workspace must be a contiguous uint8 tensor on the logits' device")
    logprobs = _output(logprobs, "logprobs", shape, torch.float32, dev)
    entropy = _output(entropy, "entropy", (R,), torch.float32, dev)
    top_ids = _output(top_ids, "top_ids", (R, top_n), torch.int32, dev)
    top_logprobs = _output(top_logprobs, "top_logprobs", (R, top_n), torch.float32, dev)
    a.abi_version, a.dtype = _abi.ABI_VERSION, dt
    a.rows, a.vocab, a.row_stride = R, V, row_stride if L > 1 else V
    a.logits = logits.data_ptr()
    a.tokens_per_row, a.top_n = K, top_n
    a.logprobs, a.entropy = logprobs.data_ptr(), entropy.data_ptr()
    a.top_ids, a.top_logprobs = top_ids.data_ptr(), top_logprobs.data_ptr()
    a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.numel()
    st = on_device(dev, lib().ecah_token_logprobs, a)
    if st:
        check(st, "ecah_token_logprobs")
    return RowLogprobs(logprobs, entropy, top_ids, top_logprobs)


def _output(t, name, shape, dtype, dev):
    if t is None:
        return torch.empty(shape, dtype=dtype, device=dev)
    n = 1
    for d in shape:
        n *= d
    _need(t, name, dtype, n, dev)
    return t


class TokenLogprobs:
    """Owns the workspace of one stream, so repeated calls (and CUDA-graph
    replays) of any number of rows allocate nothing but their outputs."""

    def __init__(self, vocab: int, dtype: torch.dtype, device="cuda"):
        if dtype not in _DTYPES:
            raise RuntimeError(f"unsupported logits dtype {dtype}")
        self.vocab, self.dtype = vocab, dtype
        self.device = resolve_device(device)
        self.workspace = new_workspace(self.device)

    def __call__(self, logits: torch.Tensor, token_ids: Optional[torch.Tensor] = None, **kw) -> RowLogprobs:
        if logits.dtype != self.dtype or logits.shape[-1] != self.vocab:
            raise RuntimeError(f"logits must be [R, {self.vocab}] {self.dtype}, "
                               f"got {list(logits.shape)} {logits.dtype}")
        return launch(logits, token_ids, self.workspace, **kw)


# ------------------------------------------------------------ torch custom op
_LIB.define(
    "token_logprobs(Tensor logits, Tensor token_ids, Tensor? temperature, Tensor? row_index, "
    "Tensor(a!) logprobs, Tensor(b!) entropy, Tensor(c!) top_ids, Tensor(d!) top_logprobs, "
    "Tensor(e!) workspace) -> ()")


def _op_cuda(logits, token_ids, temperature, row_index, logprobs, entropy, top_ids, top_logprobs, workspace):
    launch(logits, token_ids, workspace, top_n=top_ids.shape[1], temperature=temperature, row_index=row_index,
           logprobs=logprobs, entropy=entropy, top_ids=top_ids, top_logprobs=top_logprobs)


_LIB.impl("token_logprobs", _op_cuda, "CUDA")


@torch.library.register_fake("ecah::token_logprobs")
def _op_fake(logits, token_ids, temperature, row_index, logprobs, entropy, top_ids, top_logprobs, workspace):
    return None
