"""The example that prefills a prompt, forks it and verifies drafts, against a plain float32 forward;
and the manager's verification against the sampler's probabilities."""
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
    """Logits of every place of a list of tokens, all of it in float32."""
    hq, hk, dim = step.dims
    n = len(tokens)
    x = step.embed[torch.tensor(tokens, device="cuda")].float()
    c, s = step.table[:n].chunk(2, -1)
    mask = torch.ones(n, n, device="cuda").tril().bool()

    def turn(h):
        h = norm(h)
        a, b = h.chunk(2, -1)
        return torch.cat([a * c[:, None] - b * s[:, None], b * c[:, None] + a * s[:, None]], -1)

    for wqkv, wo in zip(step.wqkv, step.wo):
        qkv = (norm(x) @ wqkv.float()).view(n, hq + 2 * hk, dim)
        q, k, v = turn(qkv[:, :hq]), turn(qkv[:, hq:hq + hk]), qkv[:, hq + hk:]
        k, v = (t.repeat_interleave(hq // hk, 1) for t in (k, v))
        p = torch.einsum("ihd,jhd->hij", q, k).div(dim ** 0.5).masked_fill(~mask, float("-inf")).softmax(-1)
        x = x + torch.einsum("hij,jhd->ihd", p, v).reshape(n, -1) @ wo.float()
    return norm(x) @ step.head.float()


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("prompt", [5, 32, 41])
def test_prompt_fork_and_drafts_match_a_plain_forward(e4m3, prompt):
    """Prompts that end inside a page, and at its end; drafts of every length.  The relative errors
    that the decode step's test derives: bf16 activations through two layers, an e4m3 cache."""
    from draft_step import DraftStep
    step = DraftStep(3, 4, e4m3=e4m3, max_len=120, seed=prompt)
    most = 0.15 if e4m3 else 0.03
    g = torch.Generator().manual_seed(prompt)
    logits = step.prefill(torch.randint(0, step.vocab, (prompt,), generator=g).tolist())
    want = forward(step, step.tokens[0])
    assert float((logits.float() - want).norm() / want.norm()) < most
    for i in range(8):
        before = [list(t) for t in step.tokens]
        drafts = [torch.randint(0, step.vocab, (int(torch.randint(0, 5, (1,), generator=g)),), generator=g).tolist() for _ in before]
        if i % 2:                                        # drafts that the model itself would take
            drafts = [forward(step, t)[-1:].argmax(-1).tolist() for t in before]
        out = step(drafts)
        got = step.logits.view(3, 5, -1).float()
        for b in range(3):
            n = len(drafts[b])
            full = forward(step, before[b] + drafts[b])[-n - 1:]
            assert float((got[b, :n + 1] - full).norm() / full.norm()) < most, (i, b)
            k = int(out.accepted[b])
            assert k <= n and out.tokens[b, :k].tolist() == drafts[b][:k] and 0 <= int(out.tokens[b, k]) < step.vocab
            assert step.tokens[b] == before[b] + out.tokens[b, :k + 1].tolist()


def test_manager_verifies_against_the_sampler_s_probabilities():
    """Each row's kept set and masses by the sampler's definition, the verification by its own; greedy rows too."""
    from ecahlang_b200.drafts import verify, new_workspace
    from ecahlang_b200.manager import SamplingManager
    from ecahlang_b200.sampler import launch, new_workspace as sampler_workspace
    V, B, N = 5000, 4, 3
    m = SamplingManager(V, seq_lens=8, dtype=torch.float16, seed=3)
    m.init_sampling_buffers(8)
    m.init_draft_buffers(8, 5)
    T, K, P = [0.5, 1.0, 0.0, 2.0], [V, 40, V, 7], [0.9, 1.0, 1.0, 0.5]
    m.fill_sampling_params(B, T, K, P)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = (torch.randn(B, N + 1, V, generator=g, device="cuda") * 3).half()
    ids = x[:, :N].float().argmax(-1).int()
    ids[1, 1] = 17
    u = torch.rand(B, N + 1, generator=g, device="cuda")
    q = torch.softmax(x[:, :N].float(), -1)
    rows = lambda v, t: torch.tensor(v, dtype=t, device="cuda").repeat_interleave(N + 1)   # noqa: E731
    probs = torch.empty(B * (N + 1), V, device="cuda")
    launch(x.view(-1, V), rows(T, torch.float32), rows(K, torch.int32), rows(P, torch.float32),
           torch.empty(B * (N + 1), dtype=torch.int32, device="cuda"), sampler_workspace(B * (N + 1), V, torch.float16),
           uniforms=torch.zeros(B * (N + 1), device="cuda"), probs_out=probs)
    for draft in (None, q):
        got = m.verify_drafts(x, ids, draft, uniforms=u)
        want = verify(probs.view(B, N + 1, V), ids, u, new_workspace(B), draft_probs=draft)
        assert torch.equal(got.tokens, want.tokens) and torch.equal(got.accepted, want.accepted)
    assert got.accepted[2] == N and got.tokens[2].tolist() == x[2].float().argmax(-1).tolist()      # greedy
    a, b = (m.verify_drafts(x.view(-1, V), ids) for _ in range(2))         # the Philox offset advances
    assert int(m.philox_state[1]) == 2
    assert a.tokens.shape == (B, N + 1) and b.accepted.shape == (B,)
    m.fill_sampling_params(B, T, K, P, rep_pens=[1.2] * B, batch_ids=None)
    with pytest.raises(RuntimeError, match="penalties"):
        m.verify_drafts(x, ids)
    for change, why in ((dict(draft_ids=ids[:, :2]), "logits must be"), (dict(draft_ids=torch.zeros(9, 5, dtype=torch.int32)), "more rows"),
                        (dict(draft_ids=ids[0]), "must be")):
        with pytest.raises(RuntimeError, match=why):
            m.verify_drafts(**{**dict(logits=x, draft_ids=ids), **change})
    with pytest.raises(RuntimeError, match="init_draft_buffers"):
        SamplingManager(V, seq_lens=8, dtype=torch.float16).verify_drafts(x, ids)


def test_example_runs():
    import subprocess
    for extra in ([], ["--e4m3"]):
        out = subprocess.run([sys.executable, os.path.join(ROOT, "examples", "draft_step.py"), "--steps", "3", *extra], check=True,
                             capture_output=True, text=True).stdout
        assert out.count("step ") == 3


def test_a_captured_bucket_refuses_penalties_and_another_fill_does_not_hide_them():
    from ecahlang_b200.manager import SamplingManager
    V, B, N = 1000, 2, 3
    m = SamplingManager(V, seq_lens=8, dtype=torch.float16, seed=5)
    m.init_sampling_buffers(8)
    m.init_cuda_graph_buffers([B, 4])
    m.init_draft_buffers(8, N)
    plain = ([1.0] * B, [V] * B, [1.0] * B)
    best = torch.tensor([[7, 900, 7, 0], [999, 1, 2, 3]], device="cuda")
    x = torch.zeros(B, N + 1, V, dtype=torch.float16, device="cuda").scatter_(2, best[..., None], 9.0)
    ids = best[:, :N].int()
    m.fill_cuda_graph_sampling_params(B, B, *plain, rep_pens=[1.5] * B)
    m.fill_sampling_params(B, *plain)
    with pytest.raises(RuntimeError, match="penalties"):
        m.verify_drafts(x, ids, bucket_size=B)
    m.fill_cuda_graph_sampling_params(B, B, *plain)
    m.verify_drafts(x, ids, bucket_size=B)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m.verify_drafts(x, ids, bucket_size=B)
    for pens in (dict(rep_pens=[1.5] * B), dict(freq_pens=[0.5] * B), dict(pres_pens=[0.5] * B)):
        with pytest.raises(RuntimeError, match="captured"):
            m.fill_cuda_graph_sampling_params(B, B, *plain, **pens)
        m.fill_cuda_graph_sampling_params(4, B, *plain, **pens)
        m.fill_sampling_params(B, *plain, **pens)
    m.fill_cuda_graph_sampling_params(B, B, [0.0] * B, [V] * B, [1.0] * B)
    graph.replay()
    assert out.accepted.tolist() == [N] * B and torch.equal(out.tokens, best.int())   # greedy


def test_a_capture_survives_draft_buffers_made_again():
    from ecahlang_b200.manager import SamplingManager
    V, B, N = 3000, 2, 3
    m = SamplingManager(V, seq_lens=8, dtype=torch.float16, seed=6)
    m.init_sampling_buffers(8)
    m.init_cuda_graph_buffers([B])
    m.init_draft_buffers(B, N)
    m.fill_cuda_graph_sampling_params(B, B, [1.0] * B, [V] * B, [1.0] * B)
    g = torch.Generator(device="cuda").manual_seed(7)
    x = (torch.randn(B, N + 1, V, generator=g, device="cuda") * 3).half()
    ids, u = x[:, :N].float().argmax(-1).int(), torch.rand(B, N + 1, generator=g, device="cuda")
    m.verify_drafts(x, ids, uniforms=u, bucket_size=B)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m.verify_drafts(x, ids, uniforms=u, bucket_size=B)
    for batch, drafts in ((B, N), (4, 5)):
        m.init_draft_buffers(batch, drafts)
        junk = [torch.full((B * (N + 1) * V,), float("nan"), device="cuda") for _ in range(4)] + \
               [torch.full((n,), -7, dtype=torch.int32, device="cuda") for n in (8, 8, 2100, 4200, 8400)]
        x.copy_((torch.randn(B, N + 1, V, generator=g, device="cuda") * 3).half())
        u.copy_(torch.rand(B, N + 1, generator=g, device="cuda"))
        for _ in range(2):
            graph.replay()
            want = m.verify_drafts(x, ids, uniforms=u, bucket_size=B)
            assert torch.equal(out.tokens, want.tokens) and torch.equal(out.accepted, want.accepted)
        assert all(bool(torch.isnan(t).all()) for t in junk[:4]) and all(bool((t == -7).all()) for t in junk[4:])   # nothing in their memory
