"""Edges of the serving operators on the GPU against float64: what a wrong
answer hides behind in ordinary inputs."""
import math

import pytest
import torch

from decode_util import long_cache, long_reference
from ecahlang_b200.logprobs import TokenLogprobs, launch, new_workspace
from ecahlang_b200.manager import SamplingManager
from ecahlang_b200.paged import PagedAttention

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3 = torch.float8_e4m3fn
KINDS = [(torch.float16, None), (torch.bfloat16, None), (torch.float16, E4M3), (torch.bfloat16, E4M3)]
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}     # half a unit in the last place


@pytest.mark.parametrize("dtype,kv", KINDS)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_decode_long_tail_of_small_weights(dtype, kv, D):
    """Four dominating keys without a value and 2^15 keys at 2^-25.4 of their weight: all of the
    output comes from the tail.

    A weight's rounding: u of itself, and for f16 operands half of f16's smallest, 2^-25, with the
    largest weight at 2^7 or more: 2^-32 of the largest a key, over a sum of 4 of the largest.
    Float32's part is below 2^-16, the output's rounding u (f16: and half its smallest, 2^-25).

    1776 requests share the pages: a multiple of the blocks of 148 SMs, so that whole requests fall
    to a block, whose four warps see a dominating key each."""
    n, page, batch, gap = 1 << 15, 64, 1776, 17.625                # gap: nats; exact in 8 bits
    k = torch.zeros(n // page, page, 1, D, dtype=torch.float32, device=DEV)
    v = torch.ones_like(k)
    ks = vs = None
    k.view(n, D)[[0, 16, 32, 48], 0] = 1.0 if kv else gap
    v.view(n, D)[[0, 16, 32, 48]] = 0.0
    if kv:
        ks, vs = (torch.ones(n // page, 1, page, device=DEV) for _ in range(2))
        ks[0, 0, [0, 16, 32, 48]] = gap
    k, v = k.to(kv or dtype), v.to(kv or dtype)
    q = torch.zeros(batch, 1, D, dtype=dtype, device=DEV)
    q[:, 0, 0] = 1.0
    indptr = torch.arange(0, (batch + 1) * (n // page), n // page, dtype=torch.int32, device=DEV)
    indices = torch.arange(n // page, dtype=torch.int32, device=DEV).repeat(batch)
    last = torch.full((batch,), page, dtype=torch.int32, device=DEV)
    out, lse = PagedAttention(1, 1, D, page, dtype, kv_dtype=kv, max_batch=batch).decode(
        q, indptr, indices, last, k, v, k_scale=ks, v_scale=vs, sm_scale=1.0, return_lse=True)
    tail = (n - 4) * math.exp(-gap)
    want = tail / (4 + tail)
    weight = UNIT[torch.float16 if kv else dtype]
    tol = (UNIT[dtype] + weight + 2.0 ** -16) * want + n * 2.0 ** -32 / 4 + 2.0 ** -25
    assert float((out.double() - want).abs().max()) <= tol
    assert float((lse.double() - (gap + math.log(4 + tail))).abs().max()) <= 2e-5 + 4e-6 * gap


def _garbage_pool():
    """A graph whose memory pool holds freed blocks of a log-probability workspace's size, none of them zero."""
    graph = torch.cuda.CUDAGraph()
    n = TokenLogprobs(8, torch.float16).workspace.numel()
    with torch.cuda.graph(graph):
        kept = [torch.empty(n, dtype=torch.uint8, device=DEV).fill_(0x5A) for _ in range(12)]
    graph.replay()
    del kept
    return graph


def test_manager_calls_first_made_inside_a_capture():
    """The first `sample` and `logprobs` of a manager are captured; an eager call and another bucket
    run before that graph is replayed."""
    V = 151936
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(4, V, generator=g, device=DEV).half()
    m = SamplingManager(V, seq_lens=8, dtype=torch.float16, seed=1)
    m.init_sampling_buffers(8)
    m.init_cuda_graph_buffers([2, 4])
    for bs in (2, 4):
        m.fill_cuda_graph_sampling_params(bs, bs, [0.7] * bs, [V] * bs, [0.9] * bs)
    m.fill_sampling_params(4, [0.7] * 4, [V] * 4, [0.9] * 4)
    pool = _garbage_pool()
    got, graphs = {}, {}
    for bs in (2, 4):
        graphs[bs] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graphs[bs], pool=pool.pool()):
            ids = m.sample(x[:bs], bucket_size=bs, uniforms=torch.full((bs,), 0.5, device=DEV))
            got[bs] = m.logprobs(x[:bs], ids, 5, bucket_size=bs), ids
    want = TokenLogprobs(V, torch.float16)

    def same(rows, a, ids):
        b = want(x[:rows], ids, top_n=5)
        assert all(torch.equal(p, q) for p, q in zip(a, b))

    u = torch.full((4,), 0.5, device=DEV)
    ids = m.sample(x, uniforms=u)
    same(4, m.logprobs(x, ids, 5), ids)
    for bs in (4, 2):
        graphs[bs].replay()
        same(bs, *got[bs])
        assert torch.equal(got[bs][1], ids[:bs])


def test_manager_logprobs_takes_the_row_index_that_sample_takes():
    V = 5000
    x = torch.randn(9, V, generator=torch.Generator(device=DEV).manual_seed(4), device=DEV).half()
    m = SamplingManager(V, seq_lens=8, dtype=torch.float16, seed=1)
    m.init_sampling_buffers(8)
    m.fill_sampling_params(3, [0.5, 1.0, 2.0], [V] * 3, [0.9] * 3)
    at = torch.tensor([8, 0, 8], dtype=torch.int32, device=DEV)
    ids = m.sample(x, row_index=[8, 0, 8])
    want = TokenLogprobs(V, torch.float16)(x[at.long()], ids, top_n=3, temperature=torch.tensor([0.5, 1.0, 2.0], device=DEV))
    for rows in ([8, 0, 8], at, at.cpu(), (8, 0, 8)):
        got = m.logprobs(x, ids, 3, row_index=rows, tempered=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [7, 5000, 151936])
def test_logprobs_with_the_smallest_temperatures(dtype, V):
    """All mass is on the largest logits, evenly."""
    x = torch.zeros(3, V, dtype=dtype, device=DEV)
    x[:, 1], x[:, 3] = 2.0, 2.0
    T = torch.tensor([2.0 ** -149, 2.0 ** -148, 2.0 ** -126], device=DEV)
    tok = torch.tensor([[1, 0]] * 3, dtype=torch.int32, device=DEV)
    got = launch(x, tok, new_workspace(), top_n=3, temperature=T)
    for r in range(3):
        assert abs(float(got.logprobs[r, 0]) + math.log(2)) <= 1e-6 and float(got.logprobs[r, 1]) < -1e37
        assert abs(float(got.entropy[r]) - math.log(2)) <= 1e-6
        assert got.top_ids[r].tolist() == [1, 3, 0]
        assert (got.top_logprobs[r, :2] + math.log(2)).abs().max() <= 1e-6 and float(got.top_logprobs[r, 2]) < -1e37


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [7, 5000, 151936])
def test_logprobs_without_a_temperature(dtype, V):
    """A NaN is no temperature: its row has no distribution, the row beside it has one."""
    x = torch.zeros(2, V, dtype=dtype, device=DEV)
    x[:, 1], x[:, 3] = 2.0, 2.0
    T = torch.tensor([float("nan"), 1.0], device=DEV)
    tok = torch.tensor([[1, 0]] * 2, dtype=torch.int32, device=DEV)
    got = launch(x, tok, new_workspace(), top_n=3, temperature=T)
    assert torch.isnan(got.logprobs[0]).all() and torch.isnan(got.entropy[0]) and torch.isnan(got.top_logprobs[0]).all()
    assert got.top_ids[0].tolist() == [-1] * 3
    assert got.top_ids[1].tolist() == [1, 3, 0] and torch.isfinite(got.logprobs[1]).all()


@pytest.mark.parametrize("dtype,kv", KINDS)
@pytest.mark.parametrize("Hq,Hk,D,lengths,listed", [
    (16, 2, 128, [40000], 0), (16, 2, 128, [5, 70001, 1, 0], 0), (32, 8, 128, [40001, 33, 39000, 3001], 0),
    (40, 2, 64, [30011, 700], 0), (8, 4, 192, [25000, 9], 100_000), (34, 2, 256, [20001, 64], 100_000),
    (12, 6, 96, [1500, 35000], 100_000)])
def test_decode_long_contexts(dtype, kv, Hq, Hk, D, lengths, listed):
    """Work divided over the blocks and joined, at a tolerance that a lost run of keys exceeds."""
    g = torch.Generator(device=DEV).manual_seed(D + Hq)
    page = 16
    parts = [long_cache(n, page, Hk, D, dtype, kv is not None, g, DEV) for n in lengths if n]
    q = (torch.randn(len(lengths), Hq, D, generator=g, device=DEV) * 1.5).to(dtype)
    cat = lambda ts: torch.cat([t.view(torch.uint8) for t in ts]).view(ts[0].dtype) if ts[0] is not None else None   # noqa: E731
    k, v, ks, vs = (cat([p[i] for p in parts]) for i in range(4))
    # pages in a scattered order
    order = torch.randperm(k.shape[0], generator=g, device=DEV)
    place = torch.empty_like(order)
    place[order] = torch.arange(len(order), device=DEV)
    k, v = (c.view(torch.uint8)[order].view(c.dtype) for c in (k, v))
    if ks is not None:
        ks, vs = ks[order].contiguous(), vs[order].contiguous()
    counts = [-(-n // page) for n in lengths]
    indptr = torch.tensor([0] + counts).cumsum(0).to(torch.int32).to(DEV)
    indices = torch.cat([place.to(torch.int32), torch.zeros(listed, dtype=torch.int32, device=DEV)])
    last = torch.tensor([(n - 1) % page + 1 if n else 0 for n in lengths], dtype=torch.int32, device=DEV)
    out, lse = PagedAttention(Hq, Hk, D, page, dtype, kv_dtype=kv).decode(
        q, indptr, indices, last, k, v, k_scale=ks, v_scale=vs, return_lse=True)
    at = 0
    for b, n in enumerate(lengths):
        if not n:
            assert (out[b] == 0).all() and (lse[b] == -math.inf).all()
            continue
        want, wlse, tol = long_reference(q[b], n, *parts[at], dtype)
        at += 1
        assert ((out[b].double() - want).abs() <= tol).all(), float(((out[b].double() - want).abs() / tol).max())
        assert ((lse[b].double() - wlse).abs() <= 2e-5 + 4e-6 * 16).all()


def test_expanded_tensors_are_read_but_not_written():
    """Rows that share memory serve as inputs; as outputs, whose rows are written in no order, they are refused."""
    att = PagedAttention(8, 2, 64, 16, torch.float16, max_batch=4)
    k, v, _, _ = att.new_cache(3)
    t = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)   # noqa: E731
    one = torch.randn(1, 1, 64, device=DEV).half()
    q, new = one.expand(4, 8, 64), one.expand(4, 2, 64)
    place = (t(0, 1, 2, 3), t(0, 0, 0, 0), t(0, 1, 1, 1, 1), t(2))
    got = att.append(q, new, new, *place, k, v)
    assert torch.equal(got, q) and torch.equal(k[2, :4], new) and torch.equal(v[2, :4], new)
    for bad in (dict(q_out=torch.empty_like(one).expand(4, 8, 64)), dict(q_out=torch.empty(4, 1, 64, device=DEV).half().expand(4, 8, 64))):
        with pytest.raises(RuntimeError, match="share memory"):
            att.append(q, new, new, *place, k, v, **bad)
    for bad in ((k[:1].expand(3, 16, 2, 64), v), (k, v[:, :, :1].expand(3, 16, 2, 64)), (k[:, :1].expand(3, 16, 2, 64), v)):
        with pytest.raises(RuntimeError, match="share memory"):
            att.append(q, new, new, *place, *bad)
    last = t(4, 0, 0, 0)
    out = att.decode(q, place[2], place[3], last, k, v)
    shared = att.decode(q, place[2], place[3], last, k[:, :, :1].expand(3, 16, 2, 64), v[:, :, :1].expand(3, 16, 2, 64))
    assert torch.equal(out, shared)
    with pytest.raises(RuntimeError, match="share memory"):
        att.decode(q, place[2], place[3], last, k, v, out=torch.empty_like(one).expand(4, 8, 64))


def test_manager_keeps_the_workspace_that_a_captured_bucket_uses():
    """The sampling buffers are made again, larger, between the capture and a replay."""
    V = 151936
    x = torch.randn(2, V, generator=torch.Generator(device=DEV).manual_seed(5), device=DEV).half()
    ids = torch.tensor([7, 9], dtype=torch.int32, device=DEV)
    m = SamplingManager(V, seq_lens=8, dtype=torch.float16, seed=1)
    m.init_sampling_buffers(2)
    m.logprobs(x, ids, 5)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = m.logprobs(x, ids, 5)
    m.init_sampling_buffers(16)
    n = TokenLogprobs(8, torch.float16).workspace.numel()
    kept = [torch.empty(n, dtype=torch.uint8, device=DEV).fill_(0x5A) for _ in range(8)]
    graph.replay()
    want = TokenLogprobs(V, torch.float16)(x, ids, top_n=5)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and all((t == 0x5A).all() for t in kept)
