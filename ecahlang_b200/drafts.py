"""Verification of drafted tokens: ``DraftVerifier`` / ``verify`` and the torch
custom op ``torch.ops.ecah.verify_drafts``.

A draft (a small model, or a look-up in the prompt) proposes up to N tokens a
request; the model runs over all of them at once (``PagedAttention.prefill``),
and the verification keeps the longest run of them that leaves the output
distributed as the model's own samples, and draws the token behind it.  The
reference decodes one token a step (ecahlang/main.py:334-422).  The arithmetic
lives in ``libecah_sampler.so``; its torch binding (csrc/binding.cpp) checks
tensors and launches on the current torch stream.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from ._abi import binding, lib
from .sampler import _LIB, resolve_device


class VerifiedDrafts(NamedTuple):
    """One launch's results: request b goes on with ``tokens[b, :accepted[b] + 1]``."""
    tokens: torch.Tensor         # int32 [B, N + 1]: the kept drafts, the drawn token, then -1
    accepted: torch.Tensor       # int32 [B]: kept drafts


def new_workspace(batch: int, device="cuda") -> torch.Tensor:
    """Zero-filled workspace of launches of up to `batch` requests; one per
    stream that may run a launch concurrently."""
    return torch.zeros(int(lib().ecah_verify_drafts_workspace_bytes(batch)), dtype=torch.uint8, device=resolve_device(device))


def verify(target_probs: torch.Tensor, draft_ids: torch.Tensor, uniforms: torch.Tensor, workspace: torch.Tensor, *,
           draft_probs: Optional[torch.Tensor] = None, num_drafts: Optional[torch.Tensor] = None,
           tokens: Optional[torch.Tensor] = None, accepted: Optional[torch.Tensor] = None) -> VerifiedDrafts:
    """Enqueue one verification of ``draft_ids`` int32 [B, N].

    ``target_probs`` [B, N + 1, V] (float32, float16 or bfloat16; rows
    contiguous): the model's probabilities of the token at each place, after
    temperature, top-k and top-p -- the sampler's ``probs_out``; row j is of the
    place that draft j would take, row N of the place behind the last.
    ``draft_probs`` [B, N, V]: what each draft was drawn from (None: the drafts
    are certain, as from a look-up).  ``uniforms`` float32 [B, N + 1] in [0, 1):
    one for each draft's test, the last for the drawn token.  ``num_drafts``
    int32 [B] (None: N): request b has that many of its N places filled; -1
    marks a padding row (tokens -1, accepted 0).

    Draft j is kept while ``u q(x) < p(x)``; after the first refusal the token
    is drawn from ``max(p - q, 0)``, else from the row behind the drafts, as the
    first index whose cumulative mass exceeds ``u`` times the whole."""
    return VerifiedDrafts._make(binding().verify(target_probs, draft_ids, uniforms, workspace, draft_probs, num_drafts,
                                                 tokens, accepted, -1, -1))


class DraftVerifier:
    """Owns the workspace of one stream, so repeated calls (and CUDA-graph
    replays) of up to ``max_batch`` requests allocate nothing but their outputs."""

    def __init__(self, vocab: int, max_batch: int = 128, device="cuda"):
        if vocab < 1 or max_batch < 1:
            raise RuntimeError("vocab and max_batch must be positive")
        self.vocab, self.max_batch = vocab, max_batch
        self.device = resolve_device(device)
        self.workspace = new_workspace(max_batch, self.device)
        self._verify = binding().verify

    def __call__(self, target_probs: torch.Tensor, draft_ids: torch.Tensor, uniforms: torch.Tensor, *,
                 draft_probs: Optional[torch.Tensor] = None, num_drafts: Optional[torch.Tensor] = None,
                 tokens: Optional[torch.Tensor] = None, accepted: Optional[torch.Tensor] = None) -> VerifiedDrafts:
        """``verify`` on this handle's workspace."""
        return VerifiedDrafts._make(self._verify(target_probs, draft_ids, uniforms, self.workspace, draft_probs,
                                                 num_drafts, tokens, accepted, self.vocab, self.max_batch))


# ------------------------------------------------------------ torch custom op
_LIB.define(
    "verify_drafts(Tensor target_probs, Tensor draft_ids, Tensor uniforms, Tensor? draft_probs, Tensor? num_drafts, "
    "Tensor(a!) tokens, Tensor(b!) accepted, Tensor(c!) workspace) -> ()")


def _op_cuda(target_probs, draft_ids, uniforms, draft_probs, num_drafts, tokens, accepted, workspace):
    verify(target_probs, draft_ids, uniforms, workspace, draft_probs=draft_probs, num_drafts=num_drafts, tokens=tokens,
           accepted=accepted)


_LIB.impl("verify_drafts", _op_cuda, "CUDA")


@torch.library.register_fake("ecah::verify_drafts")
def _op_fake(target_probs, draft_ids, uniforms, draft_probs, num_drafts, tokens, accepted, workspace):
    return None
