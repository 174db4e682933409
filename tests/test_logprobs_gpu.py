"""Token log probabilities on the GPU against the definition in float64.

Tolerances, from the arithmetic: a log probability is (x - m)/T - ln Z.  Three
float32 roundings of a number of the result's size give 2^-22 of it.  Z is a
sum of V terms of at most 2^-21 relative error each (the exponent's rounding
and the exponential's), added in chains of at most V / 256 terms: at most
V / 256 * 2^-24 of Z in the worst case, 4e-5 at V = 151936; random signs keep it
under a tenth of that.  1e-5 absolute plus 2^-21 relative is used throughout.
The entropy adds the same error times the mean of |z|.
"""
import numpy as np
import pytest
import torch

from ecahlang_b200 import logprobs as L

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float16, torch.bfloat16, torch.float32]
ATOL, RTOL = 1e-5, 2.0 ** -21


def reference(x, tok, top_n, temperature=None):
    """Float64, row by row, edges included."""
    R, V = x.shape
    xd = x.double().cpu().numpy()
    T = np.ones(R) if temperature is None else temperature.double().cpu().numpy()
    tok = tok.cpu().numpy().reshape(R, -1)
    lp = np.full(tok.shape, np.nan)
    ent = np.full(R, np.nan)
    ids = np.full((R, top_n), -1)
    top = np.full((R, top_n), np.nan)
    for r in range(R):
        v = xd[r]
        if np.isnan(v).any() or np.isposinf(v).any():
            continue
        top[r] = -np.inf
        if np.isneginf(v).all():
            row, ent[r] = np.full(V, -np.inf), 0.0
        elif T[r] <= 0:
            row, ent[r] = np.full(V, -np.inf), 0.0
            row[np.argmax(v)] = 0.0
        else:
            z = (v - v.max()) / T[r]
            lz = np.log(np.exp(z).sum())
            row = z - lz
            e = np.exp(z)
            ent[r] = lz - (e[e > 0] * z[e > 0]).sum() / e.sum()
        ok = (tok[r] >= 0) & (tok[r] < V)
        lp[r, ok] = row[tok[r, ok]]
        order = np.lexsort((np.arange(V), -v))
        order = order[v[order] > -np.inf][:top_n]
        ids[r, :len(order)], top[r, :len(order)] = order, row[order]
    with np.errstate(over="ignore"):             # results are float32: past its largest they are infinite
        lp, ent, top = (v.astype(np.float32).astype(np.float64) if np.isinf(v.astype(np.float32)).any() else v
                        for v in (lp, ent, top))
    return lp, ent, ids, top


def agree(got, want):
    lp, ent, ids, top = want
    np.testing.assert_array_equal(got.top_ids.cpu().numpy(), ids)
    for g, w in ((got.logprobs, lp), (got.top_logprobs, top), (got.entropy, ent)):
        g = g.double().cpu().numpy().reshape(w.shape)
        np.testing.assert_array_equal(np.isfinite(g), np.isfinite(w))
        np.testing.assert_array_equal(np.isnan(g), np.isnan(w))
        f = np.isfinite(w)
        big = np.abs(w[f]) if w is not ent else np.full(f.sum(), 30.0) + np.abs(w[f])
        assert (np.abs(g[f] - w[f]) <= ATOL + RTOL * big).all(), np.abs(g[f] - w[f]).max()
        np.testing.assert_array_equal(g[~f & ~np.isnan(w)], w[~f & ~np.isnan(w)])


def check(x, tok, top_n, temperature=None, ws=None):
    got = L.launch(x, tok, L.new_workspace() if ws is None else ws, top_n=top_n, temperature=temperature)
    agree(got, reference(x, tok, top_n, temperature))
    return got


def make(R, V, dtype, seed=0, scale=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = (torch.randn(R, V, generator=g, device=DEV) * scale).to(dtype)
    tok = torch.randint(0, V, (R,), generator=g, device=DEV, dtype=torch.int32)
    return x, tok, g


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,V", [(1, 1), (3, 7), (2, 8), (5, 33), (1, 1000), (300, 300), (4, 4099), (40, 32003),
                                 (1, 151936), (3, 151936), (150, 50257)])
def test_sizes(dtype, R, V):
    x, tok, _ = make(R, V, dtype, seed=R + V)
    check(x, tok, min(20, V + 3, 32))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("top_n", [0, 1, 2, 31, 32])
def test_top_n_and_temperature(dtype, top_n):
    x, tok, g = make(9, 20001, dtype, seed=top_n)
    T = torch.tensor([1e-5, 0.3, 0.7, 1.0, 1.3, 5.0, 1e4, 0.0, -1.0], device=DEV)
    check(x, tok, top_n, T)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_longer_than_their_records(dtype):
    """A block's piece of the row is recorded and read again in several goes."""
    V = 6_000_011
    x, tok, _ = make(1, V, dtype, seed=9)
    check(x, tok, 20)
    check((torch.arange(V, device=DEV)[None] % 997).to(dtype), tok, 32)
    check(torch.zeros(1, V, device=DEV, dtype=dtype), tok, 32)


@pytest.mark.parametrize("dtype", DTYPES)
def test_row_starts_and_strides(dtype):
    """Rows at every offset from a 16-byte boundary; nothing outside them is read."""
    for off in range(0, 9):
        big = torch.full((6, 5200), float("nan"), device=DEV, dtype=dtype)
        x, tok, _ = make(6, 4501, dtype, seed=off)
        view = big[:, off:off + 4501]
        view.copy_(x)
        check(view, tok, 8)
        odd = torch.full((6 * 4503 + off,), float("nan"), device=DEV, dtype=dtype)
        rows = odd[off:].view(6, 4503)[:, :4501]
        rows.copy_(x)
        check(rows, tok, 8)


@pytest.mark.parametrize("dtype", DTYPES)
def test_ties_and_orders(dtype):
    """Equal values go to the lower id, however many there are and wherever the row grows."""
    V = 40001
    rows = torch.stack([
        torch.full((V,), 1.5), torch.zeros(V), torch.where(torch.arange(V) % 2 == 0, 0.0, -0.0),
        torch.linspace(-5, 5, V), torch.linspace(5, -5, V), (torch.arange(V) % 7).float(),
        (torch.arange(V) // 1000).float(), torch.where(torch.arange(V) > V - 40, 3.0, 1.0),
        torch.where(torch.arange(V) < 3, 3.0, 1.0),
        -(torch.arange(V) % 1024).float().abs(),
    ]).to(dtype).to(DEV)
    tok = torch.arange(rows.shape[0], device=DEV, dtype=torch.int32) * 11
    check(rows, tok, 32)
    check(rows, tok, 5)
    check(rows.repeat(20, 1), tok.repeat(20), 20)       # enough rows that none is split


@pytest.mark.parametrize("dtype", DTYPES)
def test_masks_infinities_and_nan(dtype):
    V = 30000
    low = torch.finfo(dtype).min
    x, tok, g = make(16, V, dtype, seed=3)
    inf = float("inf")
    x[0] = -inf                                   # nothing allowed
    x[1, 100:] = -inf                             # some allowed
    x[2] = -inf
    x[2, 29999] = 1.0                             # one allowed
    x[3, 17] = float("nan")
    x[4, 29998] = inf
    x[5, 100:] = low                              # the type's lowest value as a mask
    x[6] = low
    x[7] = low
    x[7, ::3] = -inf
    x[8] = torch.finfo(dtype).max
    x[9] = -inf
    x[9, [5, 4, 20000]] = low
    x[10, ::2] = -inf
    x[11, :] = -inf
    x[11, :9] = torch.arange(9, device=DEV).to(dtype)
    x[12] = float("nan")
    x[13, 0] = torch.finfo(dtype).max
    x[13, 1] = low
    x[14] = x[14] * 0 + 1000
    x[15] = -inf
    x[15, 12345] = float("nan")
    toks = torch.stack([tok, torch.full_like(tok, 5), torch.full_like(tok, -1), torch.full_like(tok, V)], 1)
    for T in (None, torch.full((16,), 0.7, device=DEV), torch.full((16,), 1e6, device=DEV),
              torch.full((16,), 1e-5, device=DEV), torch.zeros(16, device=DEV)):
        check(x, toks.contiguous(), 12, T)
    check(x.repeat(12, 1), toks.repeat(12, 1), 12)
    toks[:, 0], toks[:, 2] = 0, 1
    check(x, toks.contiguous(), 12, torch.full((16,), 1e6, device=DEV))


def test_workspace_serves_calls_of_any_shape_in_a_row():
    ws = L.new_workspace()
    for R, V, n, dtype in ((1, 151936, 20, torch.float16), (128, 151936, 20, torch.bfloat16), (3, 77, 5, torch.float32),
                           (1, 151936, 0, torch.bfloat16), (700, 1031, 32, torch.float16), (2, 128256, 32, torch.float32)):
        x, tok, _ = make(R, V, dtype, seed=V + n)
        check(x, tok, n, ws=ws)
        a, b = (L.launch(x, tok, ws, top_n=n) for _ in range(2))
        assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("K", [2, 33, 128, 129, 400])
@pytest.mark.parametrize("top_n", [0, 3])
def test_many_tokens_of_a_row(K, top_n):
    x, _, g = make(4, 3001, torch.bfloat16)
    tok = torch.randint(-1, 3003, (4, K), generator=g, device=DEV, dtype=torch.int32)
    check(x, tok, top_n)


def test_row_index_gathers_and_clamps():
    x, _, _ = make(11, 5003, torch.bfloat16)
    at = torch.tensor([10, 0, 3, 3, -5, 99], device=DEV, dtype=torch.int32)
    tok = torch.arange(6, device=DEV, dtype=torch.int32)
    got = L.launch(x, tok, L.new_workspace(), top_n=4, row_index=at)
    agree(got, reference(x[at.clamp(0, 10).long()], tok, 4))


def test_rows_past_32_bit_offsets():
    V = 151936
    rows = (1 << 31) // V + 5
    x = torch.empty(rows, V, dtype=torch.float16, device=DEV)
    small, tok, _ = make(3, V, torch.float16)
    at = torch.tensor([rows - 1, 0, rows - 2], device=DEV, dtype=torch.int32)
    x[at.long()] = small
    got = L.launch(x, tok, L.new_workspace(), top_n=6, row_index=at)
    agree(got, reference(small, tok, 6))


def test_stream_graph_and_op():
    x, tok, _ = make(5, 151936, torch.float16, seed=8)
    want = reference(x, tok, 7)
    h = L.TokenLogprobs(151936, torch.float16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = h(x, tok, top_n=7)
    torch.cuda.current_stream().wait_stream(side)
    agree(got, want)
    graph = torch.cuda.CUDAGraph()
    static = torch.zeros_like(x)
    with torch.cuda.graph(graph):
        got = h(static, tok, top_n=7)
    for k in range(2):
        static.copy_(x if k else x.flip(0))
        graph.replay()
    agree(got, want)
    out = [torch.empty(5, device=DEV), torch.empty(5, device=DEV), torch.empty(5, 7, dtype=torch.int32, device=DEV),
           torch.empty(5, 7, device=DEV)]
    torch.ops.ecah.token_logprobs(x, tok, None, None, *out, h.workspace)
    agree(L.RowLogprobs(*out), want)


def test_empty_and_refused():
    h = L.TokenLogprobs(100, torch.float16)
    x = torch.zeros(4, 100, dtype=torch.float16, device=DEV)
    tok = torch.zeros(4, dtype=torch.int32, device=DEV)
    assert h(x[:0], tok[:0], top_n=3).top_ids.shape == (0, 3)
    assert h(x, top_n=3).logprobs.shape == (4, 0)
    ws = h.workspace
    bad = [
        dict(logits=x, token_ids=tok.long(), workspace=ws),
        dict(logits=x, token_ids=tok[:3], workspace=ws),
        dict(logits=x, token_ids=tok, workspace=ws, top_n=33),
        dict(logits=x, token_ids=tok, workspace=ws, top_n=-1),
        dict(logits=x.double(), token_ids=tok, workspace=ws),
        dict(logits=x.t(), token_ids=torch.zeros(100, dtype=torch.int32, device=DEV), workspace=ws),
        dict(logits=x[0], token_ids=tok, workspace=ws),
        dict(logits=x, token_ids=tok.cpu(), workspace=ws),
        dict(logits=x, token_ids=tok, workspace=ws, temperature=torch.ones(3, device=DEV)),
        dict(logits=x, token_ids=tok, workspace=ws, top_ids=torch.zeros(4, 1, device=DEV), top_n=1),
        dict(logits=x, token_ids=tok, workspace=ws.float()),
        dict(logits=x, token_ids=tok, workspace=ws[:16]),
        dict(logits=x[:0], token_ids=tok[:1], workspace=ws, row_index=tok[:1]),
        dict(logits=x[:, :0], token_ids=tok, workspace=ws),
    ]
    for kw in bad:
        with pytest.raises(RuntimeError):
            L.launch(kw.pop("logits"), kw.pop("token_ids"), kw.pop("workspace"), **kw)
    with pytest.raises(RuntimeError):
        h(x[:, :50], tok)
