"""Token log probabilities: ``TokenLogprobs`` / ``launch`` and the torch custom
op ``torch.ops.ecah.token_logprobs``.

For every row of logits: the log probability of given tokens, the entropy of
the row's distribution and its most likely alternatives, in one read of the
logits -- the ``logprobs`` / ``top_logprobs`` fields of a completion, which the
reference does not offer (ecahlang/main.py:377-379 keeps the drawn id alone).
Works on a decode batch (the sampled ids) and on a prompt (every position's
next token).  The arithmetic lives in ``libecah_sampler.so``; its torch
binding (csrc/binding.cpp) checks tensors and launches on the current torch
stream.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _abi
from ._abi import binding, lib
from .sampler import _DTYPES, _LIB, resolve_device

MAX_TOP_N = _abi.MAX_TOP_N


class RowLogprobs(NamedTuple):
    """One launch's results.  ``top_ids`` is -1 (and ``top_logprobs`` -inf)
    past a row's last entry above -inf."""
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
    return RowLogprobs._make(binding().logprobs(logits, token_ids, workspace, top_n, temperature, row_index, logprobs,
                                                entropy, top_ids, top_logprobs, -1))


class TokenLogprobs:
    """Owns the workspace of one stream, so repeated calls (and CUDA-graph
    replays) of any number of rows allocate nothing but their outputs.
    ``workspace``: one that ``new_workspace`` made before (default: a new one)."""

    def __init__(self, vocab: int, dtype: torch.dtype, device="cuda", workspace: Optional[torch.Tensor] = None):
        if dtype not in _DTYPES:
            raise RuntimeError(f"unsupported logits dtype {dtype}")
        self.vocab, self.dtype = vocab, dtype
        self.device = resolve_device(device)
        self.workspace = new_workspace(self.device) if workspace is None else workspace
        self._launch = binding().logprobs

    def __call__(self, logits: torch.Tensor, token_ids: Optional[torch.Tensor] = None, *, top_n: int = 0,
                 temperature: Optional[torch.Tensor] = None, row_index: Optional[torch.Tensor] = None,
                 logprobs: Optional[torch.Tensor] = None, entropy: Optional[torch.Tensor] = None,
                 top_ids: Optional[torch.Tensor] = None, top_logprobs: Optional[torch.Tensor] = None) -> RowLogprobs:
        """``launch`` on this handle's workspace."""
        if logits.dtype is not self.dtype:
            raise RuntimeError(f"logits must be {self.dtype}, got {logits.dtype}")
        return RowLogprobs._make(self._launch(logits, token_ids, self.workspace, top_n, temperature, row_index,
                                              logprobs, entropy, top_ids, top_logprobs, self.vocab))


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
