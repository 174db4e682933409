"""Draft verification on the GPU against its definition in Python's exact arithmetic
(``fractions``) where sizes allow it, and in float64.

The kept drafts follow from exact products and are compared exactly.  The drawn
token is the first whose cumulative mass exceeds u times the whole; float64 sums
of at most V = 152 000 entries are off by less than V 2^-53 of the whole, 2e-11,
so a token is right if the target lies within its mass up to that."""
import pytest
import torch

from ecahlang_b200 import drafts
from ecahlang_b200.drafts import DraftVerifier

pytestmark = pytest.mark.gpu
DEV = "cuda"


def probs(shape, g, sharp=2.5, dtype=torch.float32, kept=1.0):
    x = torch.randn(shape, generator=g, device=DEV) * sharp
    if kept < 1.0:
        x = x.masked_fill(torch.rand(shape, generator=g, device=DEV) > kept, float("-inf"))
        x[..., :1] = 0.0
    return torch.softmax(x, -1).to(dtype)


def check(p, ids, u, q=None, num=None, got=None, slack=2e-11):
    """Every request's result against the definition, in float64 on the host."""
    B, N1, V = p.shape
    N = N1 - 1
    tokens, accepted = got.tokens.cpu(), got.accepted.cpu()
    for b in range(B):
        n = N if num is None else min(int(num[b]), N)
        row = tokens[b].tolist()
        if n < 0:
            assert row == [-1] * N1 and int(accepted[b]) == 0
            continue
        k = n
        for j in range(n):
            x = int(ids[b, j])
            if not 0 <= x < V:
                k = j
                break
            qx = 1.0 if q is None else float(q[b, j, x])
            if not float(u[b, j]) * qx < float(p[b, j, x]):
                k = j
                break
        assert int(accepted[b]) == k, (b, int(accepted[b]), k)
        assert row[:k] == ids[b, :k].tolist() and row[k + 1:] == [-1] * (N - k)
        r = p[b, k].float()
        if k < n:
            if q is not None:
                r = (r - q[b, k].float()).clamp_min(0)
            elif 0 <= int(ids[b, k]) < V:
                r = r.clone()
                r[int(ids[b, k])] = 0
        r = r.double()
        total = float(r.sum())
        if total == 0:
            r = p[b, k].double()
            total = float(r.sum())
        t = row[k]
        if not (0 < total < float("inf")):
            assert t == -1
            continue
        c = r.cumsum(0)
        target = float(u[b, N]) * total
        assert 0 <= t < V and float(r[t]) > 0
        assert float(c[t]) > target - slack * total, (b, t)
        assert float(c[t] - r[t]) <= target + slack * total, (b, t)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("V", [1, 2, 7, 255, 256, 2047, 2049, 32003, 151936])
@pytest.mark.parametrize("given", [True, False])
def test_against_the_definition(dtype, V, given):
    g = torch.Generator(device=DEV).manual_seed(V)
    B, N = 9, 4
    p = probs((B, N + 1, V), g, dtype=dtype)
    q = probs((B, N, V), g, dtype=dtype)
    q[B // 2:] = (p[B // 2:, :N].float() * 0.9).to(dtype)      # drafts that are mostly kept
    ids = torch.randint(0, V, (B, N), generator=g, device=DEV, dtype=torch.int32)
    ids[::2] = p[::2, :N].float().argmax(-1).int()
    u = torch.rand((B, N + 1), generator=g, device=DEV)
    q = q if given else None
    num = torch.tensor([4, 3, 0, -1, 2, 4, 1, 9, -7], dtype=torch.int32, device=DEV)
    ver = DraftVerifier(V, max_batch=B)
    for n in (None, num):
        check(p, ids, u, q, n, ver(p, ids, u, draft_probs=q, num_drafts=n))
    a, b = ver(p, ids, u, draft_probs=q), ver(p, ids, u, draft_probs=q)
    assert torch.equal(a.tokens, b.tokens)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_rows_and_odd_starts(dtype):
    """Rows of a wider buffer that begin on no common boundary."""
    g = torch.Generator(device=DEV).manual_seed(3)
    B, N, V = 5, 3, 5000
    big = torch.zeros((B + 1, N + 3, V + 13), dtype=dtype, device=DEV)
    big.fill_(float("nan"))
    draft = torch.full((N, B, V + 6), float("nan"), dtype=dtype, device=DEV)
    p, q = big[1:, 1:N + 2, 5:V + 5], draft.transpose(0, 1)[:, :, 1:V + 1]
    p.copy_(probs((B, N + 1, V), g, dtype=dtype))
    q.copy_(probs((B, N, V), g, dtype=dtype))
    ids = torch.randint(0, V, (B, N), generator=g, device=DEV, dtype=torch.int32)
    u = torch.rand((B, N + 1), generator=g, device=DEV)
    check(p, ids, u, q, None, DraftVerifier(V, B)(p, ids, u, draft_probs=q))
    one = p[:, :1]                                   # no drafts: a draw from the row
    check(one, ids[:, :0], u[:, :1].contiguous(), None, None, DraftVerifier(V, B)(one, ids[:, :0], u[:, :1].contiguous()))
    wide = p.expand(B, N + 1, V)[:1].expand(B, N + 1, V)      # one request's probabilities for all
    check(wide, ids, u, None, None, DraftVerifier(V, B)(wide, ids, u))


def test_edges():
    V, g = 3000, torch.Generator(device=DEV).manual_seed(5)
    p = torch.zeros((12, 2, V), device=DEV)
    q = torch.zeros((12, 1, V), device=DEV)
    ids = torch.zeros((12, 1), dtype=torch.int32, device=DEV)
    u = torch.full((12, 2), 0.5, device=DEV)
    p[0, :, 7] = 1.0; q[0, 0, 7] = 1.0; ids[0] = 7                      # sure of the same token: kept
    p[1, 0, 7] = 1.0; q[1, 0, 8] = 1.0; ids[1] = 8; p[1, 1] = 1.0 / V   # sure of another: refused, and 7
    p[2, 0, 3] = 0.5; q[2, 0, 3] = 0.5; ids[2] = 3; u[2, 0] = 0.0       # u = 0 keeps what has any mass
    p[2, 1, 2999] = 1e-30                                               # a mass far below one
    ids[3] = V; p[3, 0, 11] = 0.25                                      # outside the vocabulary: refused
    ids[4] = -1; p[4, 0, 12] = 0.25
    p[5, 0, 4] = 0.25; q[5, 0, 4] = 0.75; q[5, 0, 9] = 0.25; ids[5] = 4; u[5, 0] = 0.999   # p below q throughout: from p
    ids[6] = 1                                                          # no mass at all
    p[7, 0, 5] = float("nan"); ids[7] = 6                               # NaN in the row that is drawn from
    p[8, 0, 5] = float("inf"); ids[8] = 6
    q[9, 0, 5] = float("nan"); p[9, 0, 6] = 0.1; q[9, 0, 7] = 1.0; ids[9] = 7
    p[10, 0, 5] = 1.0; q[10, 0, 5] = 0.0; ids[10] = 5; u[10, 0] = 0.999; p[10, 1, 0] = 1.0  # q(x) = 0: kept
    p[11, 0, :] = 1.0 / V; q[11, 0, :] = 1.0 / V; ids[11] = 2; p[11, 1] = 1.0 / V; u[11, 1] = 1 - 2.0 ** -24
    got = DraftVerifier(V, 12)(p, ids, u, draft_probs=q)
    want = [[7, 7], [7, -1], [3, 2999], [11, -1], [12, -1], [4, -1], [-1, -1], [-1, -1], [-1, -1], [-1, -1], [5, 0], [2, 2999]]
    assert got.tokens.tolist() == want
    assert got.accepted.tolist() == [1, 0, 1, 0, 0, 0, 0, 0, 0, 0, 1, 1]
    # certain drafts: the entry of a refused one is left out, in a row that holds nothing else too
    p = torch.zeros((3, 2, V), device=DEV)
    p[0, 0, 7] = 0.4; p[0, 0, 9] = 0.6; p[1, 0, 7] = 0.4
    p[2, 0, 7] = 0.6; p[2, 1, 1] = 1.0
    ids = torch.full((3, 1), 7, dtype=torch.int32, device=DEV)
    got = DraftVerifier(V, 12)(p, ids, torch.full((3, 2), 0.5, device=DEV))
    assert got.tokens.tolist() == [[9, -1], [7, -1], [7, 1]] and got.accepted.tolist() == [0, 0, 1]


def test_output_is_distributed_as_the_target():
    """40 000 requests of one draft each: the first token's frequencies against the target's
    probabilities by chi-square.  11 degrees of freedom: the statistic exceeds 45 once in 10^5."""
    g = torch.Generator(device=DEV).manual_seed(7)
    V, B = 12, 40000
    p, q = probs((V,), g, 1.0), probs((V,), g, 1.0)
    ids = torch.multinomial(q, B, replacement=True, generator=g).view(B, 1).int()
    u = torch.rand((B, 2), generator=g, device=DEV)
    ver = DraftVerifier(V, max_batch=B)
    for draft in (q.expand(B, 1, V), None):
        if draft is None:
            ids = torch.randint(0, V, (B, 1), generator=g, device=DEV, dtype=torch.int32)
        got = ver(p.expand(B, 2, V), ids, u, draft_probs=draft)
        seen = torch.bincount(got.tokens[:, 0].long(), minlength=V).double()
        want = p.double() * B
        assert float(((seen - want) ** 2 / want).sum()) < 45


@pytest.mark.parametrize("N", [31, 32, 33, 100])
def test_many_drafts(N):
    g = torch.Generator(device=DEV).manual_seed(N)
    B, V = 4, 300
    p = probs((B, N + 1, V), g)
    ids = p[:, :N].argmax(-1).int()
    u = torch.rand((B, N + 1), generator=g, device=DEV) * 0.2
    u[0] = 0.0                                         # all kept
    u[1, N - 1] = 0.9999                               # the last one refused
    u[1, :N - 1] = 0.0
    check(p, ids, u, None, None, DraftVerifier(V, B)(p, ids, u))
    q = (p[:, :N] * 0.5).contiguous()
    check(p, ids, u, q, None, DraftVerifier(V, B)(p, ids, u, draft_probs=q))


def test_large_batch_and_workspace_of_a_smaller_one():
    g = torch.Generator(device=DEV).manual_seed(9)
    V, ver = 1000, DraftVerifier(1000, max_batch=600)
    for B in (600, 3, 600, 1):
        p, q = probs((B, 3, V), g), probs((B, 2, V), g)
        ids = torch.multinomial(q.view(-1, V), 1, generator=g).view(B, 2).int()
        u = torch.rand((B, 3), generator=g, device=DEV)
        check(p, ids, u, q, None, ver(p, ids, u, draft_probs=q))
    assert int(ver.workspace.view(-1, ver.workspace.numel() // 600)[:, :256].sum()) == 0


def test_captured_and_replayed_on_another_stream():
    g = torch.Generator(device=DEV).manual_seed(11)
    B, N, V = 3, 2, 20000
    ver = DraftVerifier(V, B)
    p, q = probs((B, N + 1, V), g), probs((B, N, V), g)
    ids = torch.zeros((B, N), dtype=torch.int32, device=DEV)
    num = torch.full((B,), N, dtype=torch.int32, device=DEV)
    u = torch.zeros((B, N + 1), device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ver(p, ids, u, draft_probs=q, num_drafts=num)
    side = torch.cuda.Stream()
    for i in range(4):
        p.copy_(probs((B, N + 1, V), g))
        q.copy_(probs((B, N, V), g))
        ids.copy_(torch.multinomial(q.view(-1, V), 1, generator=g).view(B, N))
        u.copy_(torch.rand((B, N + 1), generator=g, device=DEV))
        num.copy_(torch.tensor([N, i - 1, 1]))
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graph.replay()
        side.synchronize()
        check(p, ids, u, q, num, got)


def test_refusals():
    ver = DraftVerifier(100, 4)
    p, ids, u = torch.rand(2, 3, 100, device=DEV), torch.zeros(2, 2, dtype=torch.int32, device=DEV), torch.rand(2, 3, device=DEV)
    q = torch.rand(2, 2, 100, device=DEV)
    bad = [(dict(target_probs=p[:, :, :99]), "target_probs must be"), (dict(target_probs=p.double()), "unsupported dtype"),
           (dict(target_probs=p[0]), "target_probs must be"), (dict(target_probs=p.transpose(1, 2)), "target_probs must be"),
           (dict(target_probs=torch.rand(2, 100, 100, device=DEV).transpose(1, 2)[:, :3]), "contiguous"),
           (dict(target_probs=torch.rand(5, 3, 100, device=DEV)), "max_batch"), (dict(draft_ids=ids.long()), "draft_ids"),
           (dict(draft_ids=ids[:, :1]), "draft_ids"), (dict(uniforms=u[:, :2]), "uniforms"), (dict(draft_probs=q.half()), "draft_probs"),
           (dict(draft_probs=q[:, :1]), "draft_probs"), (dict(draft_probs=q.cpu()), "draft_probs"),
           (dict(num_drafts=ids), "num_drafts"), (dict(tokens=ids), "tokens"), (dict(accepted=u), "accepted")]
    for change, why in bad:
        a = dict(target_probs=p, draft_ids=ids, uniforms=u, draft_probs=None, num_drafts=None, tokens=None, accepted=None)
        with pytest.raises(RuntimeError, match=why):
            ver(**{**a, **change})
    with pytest.raises(RuntimeError, match="workspace"):
        drafts.verify(p, ids, u, ver.workspace[1:])
    with pytest.raises(RuntimeError, match="workspace"):
        drafts.verify(p, ids, u, ver.workspace[:4096])
    tokens, accepted = torch.empty(2, 3, dtype=torch.int32, device=DEV), torch.empty(2, dtype=torch.int32, device=DEV)
    torch.ops.ecah.verify_drafts(p, ids, u, q, None, tokens, accepted, ver.workspace)
    check(p, ids, u, q, None, drafts.VerifiedDrafts(tokens, accepted))
