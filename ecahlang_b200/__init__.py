"""B200-native token sampler for the ecahLang decode loop.

``sample`` / ``Sampler`` / ``torch.ops.ecah.sample`` run the fused sm_100a
kernels of ``lib/libecah_sampler.so`` (C ABI: include/ecah_sampler.h).  Around
it stand a serving step's other operators: ``TokenLogprobs`` (log
probabilities, entropy and alternatives of the logits the sampler draws from),
``PagedAttention`` (norm, rotation and write of new tokens into the paged
key-value cache, the attention of one or several new tokens that reads it, and
copies of its pages) and ``DraftVerifier`` (which drafted tokens are kept).
"""
from .drafts import DraftVerifier  # noqa: F401
from .logprobs import TokenLogprobs  # noqa: F401
from .paged import PagedAttention  # noqa: F401
from .sampler import PenaltyState, Sampler, launch, new_philox_state, new_workspace  # noqa: F401

__all__ = ["DraftVerifier", "PagedAttention", "PenaltyState", "Sampler", "TokenLogprobs", "launch", "new_philox_state", "new_workspace"]
