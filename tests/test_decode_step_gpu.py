"""The example's captured decode step against a plain float32 forward over the
same tokens, and the manager's log probabilities against its logits."""
import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "examples"))
pytestmark = pytest.mark.gpu


def norm(x):
    return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-6)


def forward(step, tokens):
    """Logits of the last of ``tokens`` [batch, n], all of it in float32."""
    hq, hk, dim = step.dims
    B, n = tokens.shape
    x = step.embed[tokens.long()].float()
    c, s = step.table[:n].chunk(2, -1)
    mask = torch.ones(n, n, device="cuda").tril().bool()

    def turn(h):
        h = norm(h)
        a, b = h.chunk(2, -1)
        return torch.cat([a * c[:, None] - b * s[:, None], b * c[:, None] + a * s[:, None]], -1)

    for wqkv, wo in zip(step.wqkv, step.wo):
        qkv = (norm(x) @ wqkv.float()).view(B, n, hq + 2 * hk, dim)
        q, k, v = turn(qkv[:, :, :hq]), turn(qkv[:, :, hq:hq + hk]), qkv[:, :, hq + hk:]
        k, v = (t.repeat_interleave(hq // hk, 2) for t in (k, v))
        p = torch.einsum("bihd,bjhd->bhij", q, k).div(dim ** 0.5).masked_fill(~mask, float("-inf")).softmax(-1)
        x = x + torch.einsum("bhij,bjhd->bihd", p, v).reshape(B, n, -1) @ wo.float()
    return norm(x[:, -1]) @ step.head.float()


@pytest.mark.parametrize("e4m3", [False, True])
def test_captured_steps_match_a_plain_forward(e4m3):
    """20 steps over a page boundary.  The step rounds every activation to bf16
    (2^-8) through two layers, and the e4m3 cache its keys and values to 2^-4: the
    logits' relative error is bounded by a few of these, 0.03 and 0.15."""
    from decode_step import DecodeStep
    step = DecodeStep(3, e4m3=e4m3, max_len=64)
    ids = torch.tensor([5, 77, 1234], dtype=torch.int32, device="cuda")
    tokens = ids[:, None].clone()
    for i in range(20):
        logits, ids, lp = step(ids)
        want = forward(step, tokens)
        rel = float((logits.float() - want).norm() / want.norm())
        assert rel < (0.15 if e4m3 else 0.03), (i, rel)
        full = torch.log_softmax(logits.double(), -1)
        assert (lp.logprobs.double() - full.gather(1, ids.long()[:, None])[:, 0]).abs().max() < 2e-5
        assert (lp.entropy.double() + (full.exp() * full).sum(-1)).abs().max() < 5e-5
        top = torch.sort(logits.float(), descending=True, stable=True, dim=-1).indices[:, :step.top_n]
        assert torch.equal(lp.top_ids.long(), top)
        ids = ids.clone()
        tokens = torch.cat([tokens, ids[:, None]], 1)


def test_manager_tempered_and_gathered():
    from ecahlang_b200.manager import SamplingManager
    m = SamplingManager(5000, seq_lens=8, dtype=torch.float16)
    m.init_sampling_buffers(8)
    m.fill_sampling_params(3, [0.5, 1.0, 2.0], [5000] * 3, [1.0] * 3)
    x = torch.randn(10, 5000, device="cuda").half()
    at = torch.tensor([9, 0, 4], dtype=torch.int32, device="cuda")
    ids = m.sample(x, row_index=at)
    T = torch.tensor([0.5, 1.0, 2.0], device="cuda", dtype=torch.float64)
    for tempered in (False, True):
        got = m.logprobs(x, ids, 3, row_index=at, tempered=tempered)
        z = x[at.long()].double() / (T[:, None] if tempered else 1.0)
        want = torch.log_softmax(z, -1).gather(1, ids.long()[:, None])[:, 0]
        assert (got.logprobs.double() - want).abs().max() < 2e-5
