"""The paged prefill attention on the GPU against its formula in float64.

Tolerance, as for decode attention: each softmax weight is rounded to the
operand type (u of itself, 2^-8 for bf16, 2^-11 for f16 and e4m3 caches, which
the model dtype's own u bounds; for f16 2^-25 of the row's largest at most),
the output once: |error| <= u |o| + u sum p|v| + 2^-24 max(p) sum|v| +
float32's 2^-16 sum p|v|.  A row without keys is exactly zero."""
import ctypes
import math

import pytest
import torch

from ecahlang_b200 import _abi, paged
from ecahlang_b200.paged import PagedAttention
from test_paged_gpu import E4M3, HALF, KINDS, cache_of, pages_for, values

pytestmark = pytest.mark.gpu
DEV = "cuda"


def reference(q, ptr, lengths, indptr, indices, k, v, ks, vs, sm_scale, causal):
    """(out, lse, tolerance of out, of lse), float64; NaN outside the requests."""
    T, Hq, D = q.shape
    Hk = k.shape[2]
    out, tol = (torch.full((T, Hq, D), float("nan"), dtype=torch.float64, device=DEV) for _ in range(2))
    lse, ltol = (torch.full((T, Hq), float("nan"), dtype=torch.float64, device=DEV) for _ in range(2))
    u, iptr = HALF[q.dtype], indptr.tolist()
    for b, n in enumerate(lengths):
        lo, hi = ptr[b], ptr[b + 1]
        if hi <= lo:
            continue
        if not n:
            out[lo:hi], tol[lo:hi], lse[lo:hi], ltol[lo:hi] = 0.0, 0.0, -math.inf, 0.0
            continue
        pg = indices[iptr[b]:iptr[b + 1]].long()
        sel = lambda c: (c.view(torch.uint8)[pg].view(E4M3) if c.dtype == E4M3 else c[pg])   # noqa: E731
        kk, vv = (values(sel(c), None if s is None else s[pg]).reshape(-1, Hk, D)[:n] for c, s in ((k, ks), (v, vs)))
        codes = sel(v).float().double().reshape(-1, Hk, D)[:n].abs().sum(0)
        for at in range(lo, hi, 256):
            end = min(at + 256, hi)
            s = torch.einsum("thgd,nhd->thgn", q[at:end].double().view(-1, Hk, Hq // Hk, D), kk) * sm_scale
            place = torch.arange(n - (hi - lo) + at - lo, n - (hi - lo) + end - lo, device=DEV)
            if causal:
                hidden = torch.arange(n, device=DEV)[None, :] > place[:, None]
                s = s.masked_fill(hidden[:, None, None, :], -math.inf)
            l = torch.logsumexp(s, -1)
            p = torch.where(torch.isinf(l)[..., None], 0.0, torch.exp(s - torch.where(torch.isinf(l), 0.0, l)[..., None]))
            w = p if vs is None else p * vs[pg].double().transpose(1, 2).reshape(-1, Hk)[:n].t()[None, :, None, :]
            o = torch.einsum("thgn,nhd->thgd", p, vv)
            mass = torch.einsum("thgn,nhd->thgd", p, vv.abs())
            seen = p.amax(-1)[..., None]
            out[at:end] = o.reshape(-1, Hq, D)
            tol[at:end] = (u * o.abs() + (u + 2.0 ** -16) * mass + 2.0 ** -24 * w.amax(-1)[..., None] * codes[None, :, None]
                           + 1e-7 * (seen > 0)).reshape(-1, Hq, D)
            lse[at:end] = l.reshape(-1, Hq)
            big = s.masked_fill(torch.isinf(s), 0.0).abs().amax(-1).reshape(-1, Hq)
            ltol[at:end] = 2e-5 + 4e-6 * big
    return out, lse, tol, ltol


def setup(new, ctx, Hq, Hk, D, page, dtype, kv=None, layout="nhd", seed=0, scale=1.5, ahead=0, behind=0, listed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    lengths = [a + b for a, b in zip(new, ctx)]
    pages, indptr, indices, last = pages_for(lengths, page, g)
    k, v, ks, vs = cache_of(pages, page, Hk, D, kv or dtype, g, layout)
    # what no request owns, or lies past its length, must not be read
    owned = torch.zeros(pages, page, dtype=torch.bool, device=DEV)
    ptr = indptr.tolist()
    for b, n in enumerate(lengths):
        if n:
            owned[indices[ptr[b]:ptr[b + 1]].long()] = True
            owned[indices[ptr[b + 1] - 1].long(), last[b]:] = False
    for c in (k, v):
        raw = c.view(torch.uint8) if c.dtype == E4M3 else c
        raw[~owned] = 0x7F if c.dtype == E4M3 else float("nan")
    if ks is not None:
        for s in (ks, vs):
            s.transpose(1, 2)[~owned] = float("nan")
    if listed:
        indices = torch.cat([indices, torch.full((listed,), -1, dtype=torch.int32, device=DEV)])
    qptr = (torch.tensor([0] + new).cumsum(0) + ahead).tolist()
    T = qptr[-1] + behind
    q = (torch.randn(T, Hq + 3, D, generator=g, device=DEV) * scale).to(dtype)
    q[:ahead] = float("nan")
    q[qptr[-1]:] = float("nan")
    q = q[:, 1:Hq + 1]                           # strided
    return dict(q=q, ptr=qptr, qo_indptr=torch.tensor(qptr, dtype=torch.int32, device=DEV), lengths=lengths, indptr=indptr,
                indices=indices, last=last, k=k, v=v, ks=ks, vs=vs)


def call(att, s, **kw):
    return att.prefill(s["q"], s["qo_indptr"], s["indptr"], s["indices"], s["last"], s["k"], s["v"], k_scale=s["ks"],
                       v_scale=s["vs"], **kw)


def compare(s, out, lse, causal=True, sm_scale=None):
    D = s["q"].shape[2]
    want, wlse, tol, ltol = reference(s["q"], s["ptr"], s["lengths"], s["indptr"], s["indices"], s["k"], s["v"], s["ks"], s["vs"],
                                      sm_scale or 1 / math.sqrt(D), causal)
    lo, hi = s["ptr"][0], s["ptr"][-1]
    err = (out.double() - want).abs()[lo:hi]
    assert torch.isfinite(out[lo:hi]).all()
    assert (err <= tol[lo:hi]).all(), float((err / tol[lo:hi].clamp_min(1e-30)).max())
    empty = torch.isinf(wlse[lo:hi])
    assert torch.equal(torch.isneginf(lse[lo:hi]), empty)
    assert ((lse.double() - wlse).abs()[lo:hi][~empty] <= ltol[lo:hi][~empty]).all()


def check(new, ctx, Hq, Hk, D, page, dtype, kv=None, causal=True, sm_scale=None, **kw):
    s = setup(new, ctx, Hq, Hk, D, page, dtype, kv, **kw)
    att = PagedAttention(Hq, Hk, D, page, dtype, kv_dtype=kv, max_batch=len(new))
    T = s["q"].shape[0]
    out = torch.full((T, Hq + 1, D), 7.0, dtype=dtype, device=DEV)
    lse = torch.full((T, Hq), 7.0, device=DEV)
    got = call(att, s, causal=causal, sm_scale=sm_scale, out=out[:, 1:], lse=lse)
    assert got.data_ptr() == out[:, 1:].data_ptr()
    compare(s, got, lse, causal, sm_scale)
    lo, hi = s["ptr"][0], s["ptr"][-1]
    for t in (out[:lo], out[hi:], out[:, 0], lse[:lo], lse[hi:]):          # nothing else is written
        assert bool((t == 7.0).all())
    again, l2 = call(att, s, causal=causal, sm_scale=sm_scale, return_lse=True)
    assert torch.equal(again[lo:hi], got[lo:hi]) and torch.equal(l2[lo:hi], lse[lo:hi])
    return att, s


@pytest.mark.parametrize("dtype,kv", KINDS)
@pytest.mark.parametrize("D", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_head_dims(dtype, kv, D, causal):
    check([1, 0, 17, 130, 300, 3, 64], [0, 5, 0, 1, 77, 700, 128], 8, 2, D, 16, dtype, kv, causal, seed=D)


@pytest.mark.parametrize("dtype,kv", KINDS)
@pytest.mark.parametrize("heads", [(16, 2), (32, 8), (14, 2), (28, 4), (8, 8), (40, 2), (5, 1), (1, 1), (130, 1)])
def test_groups(dtype, kv, heads):
    check([5, 33, 129, 1, 0], [40, 0, 300, 999, 0], *heads, 64, 16, dtype, kv, seed=heads[0])


@pytest.mark.parametrize("dtype,kv", [(torch.bfloat16, None), (torch.float16, E4M3)])
@pytest.mark.parametrize("page", [1, 3, 16, 64, 200])
@pytest.mark.parametrize("layout", ["nhd", "hnd", "paired"])
def test_pages_and_layouts(dtype, kv, page, layout):
    check([200, 1, 40], [3, 513, 90], 8, 2, 128, page, dtype, kv, layout=layout, seed=page, listed=9)


@pytest.mark.parametrize("dtype,kv", KINDS)
@pytest.mark.parametrize("n", [1, 2, 15, 16, 31, 32, 33, 63, 64, 127, 128, 129, 255, 256, 257, 511])
def test_one_prompt_of_every_length(dtype, kv, n):
    """Around the edges of tiles of queries and keys."""
    check([n], [0], 4, 2, 128, 16, dtype, kv, seed=n)
    check([1], [n], 4, 2, 128, 16, dtype, kv, seed=n)
    check([n], [n % 130], 4, 2, 128, 16, dtype, kv, causal=False, seed=n)


@pytest.mark.parametrize("dtype,kv", KINDS)
def test_padding_rows_before_and_behind(dtype, kv):
    check([0, 9, 0, 70, 0], [0, 0, 31, 5, 0], 8, 2, 128, 16, dtype, kv, ahead=6, behind=50)


@pytest.mark.parametrize("dtype,kv", KINDS)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_tokens_that_see_no_key(dtype, kv, D):
    """More new tokens than cached ones (a cache that was cut short), and requests without pages."""
    s = setup([40, 20, 300], [0, 0, 0], 8, 2, D, 16, dtype, kv)
    s["last"] = s["last"].clone()
    # request 0 keeps 2 of its 3 pages, request 1 none, request 2 one token of its first page
    a = s["indptr"].tolist()
    keep = list(range(a[0], a[0] + 2)) + [a[2]]
    s["indices"] = s["indices"][keep]
    s["indptr"] = torch.tensor([0, 2, 2, 3], dtype=torch.int32, device=DEV)
    s["last"] = torch.tensor([5, 0, 1], dtype=torch.int32, device=DEV)
    s["lengths"] = [21, 0, 1]
    att = PagedAttention(8, 2, D, 16, dtype, kv_dtype=kv, max_batch=3)
    out, lse = call(att, s, return_lse=True)
    compare(s, out, lse)
    assert bool((out[:19] == 0).all()) and bool((out[40:359] == 0).all()) and bool((out[359] != 0).any())
    out, lse = call(att, s, return_lse=True, causal=False)
    compare(s, out, lse, causal=False)


@pytest.mark.parametrize("dtype,kv", KINDS)
def test_drafts_over_long_contexts(dtype, kv):
    check([5] * 6, [0, 30000, 17, 4000, 127, 9000], 32, 8, 128, 16, dtype, kv, seed=3)


@pytest.mark.parametrize("dtype,kv", [(torch.bfloat16, None), (torch.float16, None), (torch.bfloat16, E4M3)])
def test_a_chunk_behind_a_long_context(dtype, kv):
    check([700], [20000], 8, 1, 128, 16, dtype, kv, seed=4)
    check([64], [40000], 8, 2, 64, 16, dtype, kv, seed=5)
    check([100], [9000], 8, 2, 256, 16, dtype, kv, seed=6)


@pytest.mark.parametrize("dtype,kv", [(torch.bfloat16, None), (torch.float16, E4M3)])
def test_one_long_prompt(dtype, kv):
    check([3001], [0], 16, 2, 128, 16, dtype, kv, seed=5)


@pytest.mark.parametrize("dtype,kv", KINDS)
def test_many_requests(dtype, kv):
    g = torch.Generator().manual_seed(6)
    new = torch.randint(0, 60, (300,), generator=g).tolist()
    ctx = torch.randint(0, 200, (300,), generator=g).tolist()
    check(new, ctx, 8, 2, 64, 16, dtype, kv, seed=7)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_agrees_with_decode_on_one_token_a_request(dtype):
    s = setup([1] * 5, [0, 17, 300, 1000, 5000], 16, 2, 128, 16, dtype)
    att = PagedAttention(16, 2, 128, 16, dtype, max_batch=5)
    out, lse = call(att, s, return_lse=True)
    dec, dlse = att.decode(s["q"], s["indptr"], s["indices"], s["last"], s["k"], s["v"], return_lse=True)
    compare(s, out, lse)
    compare(s, dec, dlse)


@pytest.mark.parametrize("dtype,kv", KINDS)
@pytest.mark.parametrize("scale", [1e-4, 12.0])
def test_score_ranges(dtype, kv, scale):
    """Scores near zero, and up to hundreds: references that move often, weights that underflow."""
    check([150, 40], [200, 700], 8, 2, 128, 16, dtype, kv, scale=scale, seed=8)


@pytest.mark.parametrize("dtype,kv", KINDS)
def test_rising_scores_move_the_reference_every_tile(dtype, kv):
    """Keys whose scores grow with their place by more than a factor of 2^8 in weight a tile."""
    s = setup([300], [900], 4, 2, 64, 16, dtype, kv, seed=9)
    n, page = s["lengths"][0], 16
    j = torch.arange(n, device=DEV, dtype=torch.float32)
    pg = s["indices"][:s["indptr"][1]].long()
    rise = (j / 128 * 10).floor()
    q = torch.zeros_like(s["q"])
    q[..., 0] = 1.0
    s["q"] = q
    for i in range(n):
        row = s["k"].view(torch.uint8) if kv else s["k"]
        where = (pg[i // page], i % page)
        new = torch.zeros(2, 64, device=DEV)
        new[:, 0] = 1.0 if kv else rise[i]
        row[where] = new.to(kv or dtype).view(torch.uint8) if kv else new.to(dtype)
        if kv:
            s["ks"][where[0], :, where[1]] = rise[i]
    att = PagedAttention(4, 2, 64, 16, dtype, kv_dtype=kv, max_batch=1)
    out, lse = call(att, s, return_lse=True, sm_scale=1.0)
    compare(s, out, lse, sm_scale=1.0)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_e4m3_scales_of_every_size(D):
    """Value scales from 1e-8 to 1e4 within one request: weights carry them."""
    for dtype in (torch.float16, torch.bfloat16):
        s = setup([70, 3], [100, 1200], 8, 2, D, 16, dtype, E4M3, seed=10)
        g = torch.Generator(device=DEV).manual_seed(1)
        s["vs"].copy_(10.0 ** (torch.rand(s["vs"].shape, generator=g, device=DEV) * 6 - 5))
        att = PagedAttention(8, 2, D, 16, dtype, kv_dtype=E4M3, max_batch=2)
        pg = s["indices"].long()
        raw = s["v"].view(torch.uint8)
        for i, (a, b) in enumerate(((0, int(s["indptr"][1])), (int(s["indptr"][1]), int(s["indptr"][2])))):
            raw[pg[b - 1], int(s["last"][i]):] = 0x7F
            s["vs"][pg[b - 1], :, int(s["last"][i]):] = float("nan")
        out, lse = call(att, s, return_lse=True)
        compare(s, out, lse)


@pytest.mark.parametrize("dtype,kv", KINDS)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_nan_reaches_the_rows_that_see_it_alone(dtype, kv, D):
    s = setup([200], [0], 4, 2, D, 16, dtype, kv, seed=11)
    pg, at = int(s["indices"][150 // 16]), 150 % 16
    (s["v"].view(torch.uint8) if kv else s["v"])[pg, at, 0, 3] = 0x7F if kv else float("nan")
    att = PagedAttention(4, 2, D, 16, dtype, kv_dtype=kv, max_batch=1)
    out = call(att, s)
    bad = torch.isnan(out)
    # a value's NaN is the column's, in all rows of its tile that are computed with it: rows that
    # see the key have it, rows of requests and heads apart do not
    assert bool(bad[150:, :2, 3].all())
    assert not bool(bad[:, 2:].any()) and not bool(bad[..., :3].any()) and not bool(bad[..., 4:].any())


def test_captured_and_replayed_with_other_lengths():
    """One capture serves later batches: lengths, pages and the split of the tokens are read on the device."""
    Hq, Hk, D, page = 16, 2, 128, 16
    att = PagedAttention(Hq, Hk, D, page, torch.bfloat16, max_batch=4)
    pages, T = 400, 600
    g = torch.Generator(device=DEV).manual_seed(12)
    k, v, _, _ = cache_of(pages, page, Hk, D, torch.bfloat16, g)
    q = torch.randn(T, Hq, D, generator=g, device=DEV).bfloat16()
    qptr, indptr = torch.zeros(5, dtype=torch.int32, device=DEV), torch.zeros(5, dtype=torch.int32, device=DEV)
    indices, last = torch.zeros(pages, dtype=torch.int32, device=DEV), torch.zeros(4, dtype=torch.int32, device=DEV)
    out = torch.empty_like(q)
    lse = torch.empty(T, Hq, device=DEV)
    run = lambda: att.prefill(q, qptr, indptr, indices, last, k, v, out=out, lse=lse)   # noqa: E731
    run()
    graphs = []
    for _ in range(2):                           # two captures that share the handle's workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
        graphs.append(graph)
    for i, (new, ctx) in enumerate((([600, 0, 0, 0], [0, 0, 0, 0]), ([5, 5, 5, 5], [1000, 10, 2000, 0]), ([1, 300, 0, 7], [60, 0, 9, 700]),
                                    ([0, 0, 0, 0], [0, 0, 0, 0]))):
        lengths = [a + b for a, b in zip(new, ctx)]
        used, ip, ix, la = pages_for(lengths, page, g)
        qptr.copy_(torch.tensor([0] + new).cumsum(0))
        indptr.copy_(ip); indices[:ix.numel()] = ix; last.copy_(la)
        out.fill_(7.0); lse.fill_(7.0)
        graphs[i % 2].replay()
        s = dict(q=q, ptr=qptr.tolist(), lengths=lengths, indptr=ip, indices=ix, last=la, k=k, v=v, ks=None, vs=None)
        if sum(new):
            compare(s, out, lse)
        assert bool((out[sum(new):] == 7.0).all()) and bool((lse[sum(new):] == 7.0).all())


def test_on_another_stream():
    s = setup([300, 20], [0, 800], 8, 2, 128, 16, torch.float16, seed=13)
    att = PagedAttention(8, 2, 128, 16, torch.float16, max_batch=2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out, lse = call(att, s, return_lse=True)
    side.synchronize()
    compare(s, out, lse)


def test_split_of_one_prompt_into_chunks_gives_the_same_rows():
    """A prompt at once, and in chunks behind the context of the earlier ones."""
    s = setup([500], [0], 16, 2, 128, 16, torch.float16, seed=14)
    att = PagedAttention(16, 2, 128, 16, torch.float16, max_batch=1)
    whole, lse = call(att, s, return_lse=True)
    compare(s, whole, lse)
    for at, end in ((0, 100), (100, 101), (101, 400), (400, 500)):
        n = -(-end // 16)
        part = dict(s, q=s["q"][at:end], ptr=[0, end - at], lengths=[end], indices=s["indices"][:n])
        part["qo_indptr"] = torch.tensor([0, end - at], dtype=torch.int32, device=DEV)
        part["indptr"] = torch.tensor([0, n], dtype=torch.int32, device=DEV)
        part["last"] = torch.tensor([(end - 1) % 16 + 1], dtype=torch.int32, device=DEV)
        out, lse = call(att, part, return_lse=True)
        compare(part, out, lse)


def test_refusals():
    s = setup([4, 4], [9, 0], 8, 2, 64, 16, torch.float16)
    att = PagedAttention(8, 2, 64, 16, torch.float16, max_batch=2)
    ok = dict(q=s["q"], qo_indptr=s["qo_indptr"], kv_indptr=s["indptr"], kv_indices=s["indices"], kv_last_page_len=s["last"],
              k_cache=s["k"], v_cache=s["v"])
    one = torch.zeros(1, dtype=torch.int32, device=DEV)
    bad = [(dict(q=s["q"].bfloat16()), "cache must be|model dtype"), (dict(q=s["q"].float()), "unsupported dtype"), (dict(q=s["q"][:, :7]), "q must be"),
           (dict(q=s["q"][0]), "q must be"), (dict(q=s["q"][:, :, :32]), "q|head_dim"), (dict(qo_indptr=s["qo_indptr"].long()), "qo_indptr"),
           (dict(qo_indptr=one), "qo_indptr"), (dict(kv_indptr=one), "qo_indptr"), (dict(kv_last_page_len=one), "kv_last_page_len"),
           (dict(kv_indices=s["indices"].long()), "kv_indices"), (dict(out=torch.empty(3, 8, 64, dtype=torch.float16, device=DEV)), "out"),
           (dict(out=torch.empty(8, 8, 64, dtype=torch.float32, device=DEV)), "out"),
           (dict(out=torch.empty(1, 8, 64, dtype=torch.float16, device=DEV).expand(8, 8, 64)), "share memory"),
           (dict(lse=torch.empty(8, 7, device=DEV)), "lse"), (dict(sm_scale=0.0), "sm_scale"), (dict(sm_scale=float("inf")), "sm_scale"),
           (dict(k_cache=s["k"][:, :8]), "cache"), (dict(k_scale=torch.ones(1, device=DEV)), "no scales"),
           (dict(qo_indptr=torch.zeros(4, dtype=torch.int32, device=DEV), kv_indptr=torch.zeros(4, dtype=torch.int32, device=DEV),
                 kv_last_page_len=torch.zeros(3, dtype=torch.int32, device=DEV)), "max_batch")]
    for change, why in bad:
        with pytest.raises(RuntimeError, match=why):
            att.prefill(**{**ok, **change})
    with pytest.raises(RuntimeError, match="workspace"):
        paged.prefill(**ok, workspace=att.prefill_workspace[1:])
    with pytest.raises(RuntimeError, match="workspace"):
        paged.prefill(**ok, workspace=att.prefill_workspace[:16])
    out, lse = torch.empty_like(s["q"].contiguous()), torch.empty(8, 8, device=DEV)
    torch.ops.ecah.paged_prefill(s["q"], s["qo_indptr"], s["indptr"], s["indices"], s["last"], s["k"], s["v"], None, None, True,
                                 0.125, out, lse, att.prefill_workspace)
    compare(s, out, lse)
    assert call(att, dict(s, q=s["q"][:0])).shape == (0, 8, 64)           # no tokens: qo_indptr is clamped


@pytest.mark.parametrize("dtype,kv", KINDS)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_a_wait_that_runs_out_gives_nan_and_ends(dtype, kv, D):
    """No wait between a block's warps is given any time: every row with keys is NaN, rows without are
    zeros or NaN, no other row is written, and the next launch on the same workspace is right."""
    Hq, Hk, page = 8, 2, 16
    s = setup([300, 5, 40], [0, 6000, 2000], Hq, Hk, D, page, dtype, kv, behind=3)
    att = PagedAttention(Hq, Hk, D, page, dtype, kv_dtype=kv, max_batch=3)
    T = s["q"].shape[0]
    out, lse = torch.full((T, Hq, D), 7.0, dtype=dtype, device=DEV), torch.full((T, Hq), 7.0, device=DEV)
    q, k, v = s["q"], s["k"], s["v"]
    ptr = lambda t: None if t is None else t.data_ptr()   # noqa: E731
    a = _abi.PrefillArgs(abi_version=_abi.ABI_VERSION, dtype=0 if dtype == torch.float16 else 1, tokens=T, num_qo_heads=Hq,
                         sm_scale=D ** -0.5, causal=1, q=ptr(q), q_token_stride=q.stride(0), q_head_stride=q.stride(1), out=ptr(out),
                         out_token_stride=out.stride(0), out_head_stride=out.stride(1), lse=ptr(lse), qo_indptr=ptr(s["qo_indptr"]),
                         kv_last_page_len=ptr(s["last"]), workspace=ptr(att.prefill_workspace), workspace_bytes=att.prefill_workspace.numel())
    a.cache = _abi.KVCache(kv_dtype=_abi.KV_E4M3 if kv else a.dtype, num_pages=k.shape[0], page_size=page, num_kv_heads=Hk, head_dim=D,
                           batch=3, k_cache=ptr(k), v_cache=ptr(v), k_page_stride=k.stride(0), k_slot_stride=k.stride(1),
                           k_head_stride=k.stride(2), v_page_stride=v.stride(0), v_slot_stride=v.stride(1), v_head_stride=v.stride(2),
                           k_scale=ptr(s["ks"]), v_scale=ptr(s["vs"]), kv_indptr=ptr(s["indptr"]), kv_indices=ptr(s["indices"]),
                           num_indices=s["indices"].numel())
    stream = torch.cuda.current_stream().cuda_stream
    assert _abi.lib().ecah_paged_prefill_bounded(ctypes.byref(a), 0, stream) == 0
    torch.cuda.synchronize()
    hi = s["ptr"][-1]
    assert torch.isnan(out[:hi]).all() and torch.isnan(lse[:hi]).all()
    assert bool((out[hi:] == 7.0).all()) and bool((lse[hi:] == 7.0).all())
    assert _abi.lib().ecah_paged_prefill_bounded(ctypes.byref(a), 1 << 20, stream) == 0
    compare(s, out, lse)


@pytest.mark.parametrize("dtype,kv", KINDS)
def test_scores_far_below_zero(dtype, kv):
    """All scores near -600 (log2 units: -866): weights go by the largest, not by zero."""
    s = setup([140], [150], 4, 2, 64, 16, dtype, kv, seed=15)
    q = torch.zeros_like(s["q"])
    q[..., 0] = -20.0
    s["q"] = q
    if kv:
        s["k"].view(torch.uint8)[...] = torch.tensor(30.0, device=DEV).to(E4M3).view(torch.uint8)
        s["ks"].fill_(1.0)
    else:
        s["k"][..., 0] = 30.0 + torch.rand(s["k"].shape[:-1], device=DEV).to(dtype)
    pg, last = s["indices"].long(), int(s["last"][0])
    if not kv:
        s["k"][pg[-1], last:] = float("nan")
    att = PagedAttention(4, 2, 64, 16, dtype, kv_dtype=kv, max_batch=1)
    out, lse = call(att, s, return_lse=True, sm_scale=1.0)
    compare(s, out, lse, sm_scale=1.0)
    assert float(lse.max()) < -500


@pytest.mark.parametrize("dtype,kv", KINDS)
def test_first_keys_without_mass(dtype, kv):
    """Scores of -inf through the first two tiles of keys: no reference yet where the others begin, at -200."""
    s = setup([130], [300], 4, 2, 64, 16, dtype, kv, seed=16)
    q = torch.zeros_like(s["q"])
    q[..., 0] = 1.0
    s["q"] = q
    pg = s["indices"].long()
    n, last = s["lengths"][0], int(s["last"][0])
    if kv:
        s["k"].view(torch.uint8)[...] = torch.tensor(-1.0, device=DEV).to(E4M3).view(torch.uint8)
        s["ks"].fill_(200.0)
        s["ks"][pg[:16]] = float("inf")
        s["ks"].transpose(1, 2)[pg[-1], last:] = float("nan")
    else:
        s["k"][...] = -200.0
        s["k"][pg[:16]] = 0.0
        s["k"][pg[:16], :, :, 0] = float("-inf")
        s["k"][pg[-1], last:] = float("nan")
    att = PagedAttention(4, 2, 64, 16, dtype, kv_dtype=kv, max_batch=1)
    out, lse = call(att, s, return_lse=True, sm_scale=1.0)
    kk = -torch.full((n,), 200.0, dtype=torch.float64, device=DEV)
    kk[:256] = -math.inf
    rows = torch.arange(n - 130, n, device=DEV)
    vv = values(s["v"].view(torch.uint8)[pg].view(E4M3) if kv else s["v"][pg], None if not kv else s["vs"][pg]).reshape(-1, 2, 64)[:n]
    p = torch.softmax(kk[None, :].expand(130, n).masked_fill(torch.arange(n, device=DEV)[None, :] > rows[:, None], -math.inf), -1)
    want = torch.einsum("tn,nhd->thd", p, vv).repeat_interleave(2, 1)
    mass = torch.einsum("tn,nhd->thd", p, vv.abs()).repeat_interleave(2, 1)
    u = HALF[dtype]
    assert torch.isfinite(out).all()
    assert ((out.double() - want).abs() <= u * want.abs() + (u + 2.0 ** -16) * mass + 1e-7).all()
    assert float((lse.double() - (-200 + (rows - 255).double().log())[:, None]).abs().max()) < 1e-3


@pytest.mark.parametrize("dtype,kv", [(torch.float16, None), (torch.bfloat16, E4M3)])
def test_a_cache_without_pages(dtype, kv):
    """No key anywhere: zeros and -inf."""
    att = PagedAttention(4, 2, 64, 16, dtype, kv_dtype=kv, max_batch=2)
    k, v, ks, vs = att.new_cache(0)
    q = torch.randn(9, 4, 64, device=DEV).to(dtype)
    zero = torch.zeros(3, dtype=torch.int32, device=DEV)
    out, lse = att.prefill(q, torch.tensor([0, 4, 9], dtype=torch.int32, device=DEV), zero, zero[:0], zero[:2], k, v, k_scale=ks,
                           v_scale=vs, return_lse=True)
    assert bool((out == 0).all()) and bool(torch.isneginf(lse).all())


@pytest.mark.parametrize("kv", [None, E4M3])
@pytest.mark.parametrize("page", [16, 3])
def test_pages_past_2_to_the_31_elements(kv, page):
    """Offsets beyond 32 bits in elements and bytes, by the copy engine and by threads."""
    Hk, D = 8, 128
    pages = (5 << 30) // (page * Hk * D)
    g = torch.Generator(device=DEV).manual_seed(17)
    raw = torch.uint8 if kv else torch.bfloat16
    k, v = (torch.empty((pages, page, Hk, D), dtype=raw, device=DEV) for _ in range(2))
    ks = vs = None
    new, ctx = [40, 130], [300, 0]
    lengths = [340, 130]
    counts = [-(-n // page) for n in lengths]
    indices = (pages - 1 - torch.randperm(sum(counts) * 2, generator=g, device=DEV)[:sum(counts)]).to(torch.int32)
    at = indices.long()
    if kv:
        ks, vs = (torch.empty((pages, Hk, page), device=DEV) for _ in range(2))
        for c, s in ((k, ks), (v, vs)):
            c[at] = (torch.randn((len(at), page, Hk, D), generator=g, device=DEV) * 100).clamp(-448, 448).to(E4M3).view(torch.uint8)
            s[at] = torch.rand((len(at), Hk, page), generator=g, device=DEV) * 0.02 + 1e-3
        k, v = k.view(E4M3), v.view(E4M3)
    else:
        for c in (k, v):
            c[at] = torch.randn((len(at), page, Hk, D), generator=g, device=DEV).to(raw)
    s = dict(q=torch.randn(170, 16, D, generator=g, device=DEV).bfloat16(), ptr=[0, 40, 170], lengths=lengths,
             qo_indptr=torch.tensor([0, 40, 170], dtype=torch.int32, device=DEV),
             indptr=torch.tensor([0, counts[0], sum(counts)], dtype=torch.int32, device=DEV), indices=indices,
             last=torch.tensor([(n - 1) % page + 1 for n in lengths], dtype=torch.int32, device=DEV), k=k, v=v, ks=ks, vs=vs)
    att = PagedAttention(16, Hk, D, page, torch.bfloat16, kv_dtype=kv, max_batch=2)
    out, lse = call(att, s, return_lse=True)
    compare(s, out, lse)


def test_requests_that_overlap_are_harmless():
    """qo_indptr that decreases: not an order the contract allows, but nothing outside out is written and the
    next launch is right."""
    s = setup([50, 20], [0, 900], 8, 2, 128, 16, torch.bfloat16, seed=18)
    att = PagedAttention(8, 2, 128, 16, torch.bfloat16, max_batch=2)
    out = torch.full((72, 8, 128), 7.0, dtype=torch.bfloat16, device=DEV)
    call(att, dict(s, qo_indptr=torch.tensor([60, 10, 70], dtype=torch.int32, device=DEV)), out=out[1:71])
    assert bool((out[0] == 7.0).all()) and bool((out[71] == 7.0).all())
    got, lse = call(att, s, return_lse=True)
    compare(s, got, lse)


@pytest.mark.parametrize("dtype,kv", KINDS)
@pytest.mark.parametrize("jump", [100.0, 400.0, 30000.0, float("nan")])
def test_one_key_that_outweighs_all_before_in_every_place(dtype, kv, jump):
    """128 requests; request i's key 128 + i alone scores `jump` above the zeros before and behind it (a NaN:
    makes its rows NaN), in a tile behind the first, in every column of it."""
    B, D, page, n = 128, 64, 16, 384
    k = torch.zeros(B * n // page, page, 1, D, device=DEV)
    v = torch.zeros_like(k)
    at = torch.arange(B, device=DEV) * n + 128 + torch.arange(B, device=DEV)
    k.view(-1, D)[at, 0] = 1.0 if kv else jump
    v.view(-1, D)[at] = 3.0
    ks = vs = None
    if kv:
        ks, vs = (torch.ones(B * n // page, 1, page, device=DEV) for _ in range(2))
        ks.view(-1)[at] = jump
    q = torch.zeros(2 * B, 1, D, dtype=dtype, device=DEV)
    q[:, 0, 0] = 1.0
    att = PagedAttention(1, 1, D, page, dtype, kv_dtype=kv, max_batch=B)
    out, lse = att.prefill(q, torch.arange(0, 2 * B + 1, 2, dtype=torch.int32, device=DEV),
                           torch.arange(0, B * n // page + 1, n // page, dtype=torch.int32, device=DEV),
                           torch.arange(B * n // page, dtype=torch.int32, device=DEV), torch.full((B,), page, dtype=torch.int32, device=DEV),
                           k.to(kv or dtype), v.to(kv or dtype), k_scale=ks, v_scale=vs, sm_scale=1.0, return_lse=True)
    if math.isnan(jump):
        assert torch.isnan(out).all() and torch.isnan(lse).all()
        return
    assert bool((out == 3.0).all())
    want = jump if kv else float(torch.tensor(jump).to(dtype))
    assert float((lse - want).abs().max()) <= 2e-5 + 4e-6 * jump


def test_two_handles_on_two_streams_at_once():
    """Launches that overlap, of one kernel and of others, with a workspace each: the results of one after another."""
    from ecahlang_b200.drafts import DraftVerifier
    sets = [setup([400, 30, 7], [50, 3000, 900], 16, 2, 128, 16, torch.bfloat16, seed=20),
            setup([90, 5, 5, 5], [0, 5000, 100, 2000], 32, 8, 64, 16, torch.float16, E4M3, seed=21)]
    atts = [PagedAttention(16, 2, 128, 16, torch.bfloat16, max_batch=4), PagedAttention(32, 8, 64, 16, torch.float16, kv_dtype=E4M3, max_batch=4)]
    g = torch.Generator(device=DEV).manual_seed(22)
    p = torch.softmax(torch.randn(4, 3, 30000, generator=g, device=DEV), -1)
    ids, u = p[:, :2].argmax(-1).int(), torch.rand(4, 3, generator=g, device=DEV)
    vers = [DraftVerifier(30000, 4), DraftVerifier(30000, 4)]
    want = [call(a, s, return_lse=True) for a, s in zip(atts, sets)]
    drawn = vers[0](p, ids, u)
    streams = [torch.cuda.Stream() for _ in atts]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(25):
        for i, (a, s, st) in enumerate(zip(atts, sets, streams)):
            with torch.cuda.stream(st):
                got[i].append((*call(a, s, return_lse=True), *vers[i](p, ids, u)))
    torch.cuda.synchronize()
    for i, runs in enumerate(got):
        lo, hi = sets[i]["ptr"][0], sets[i]["ptr"][-1]
        for out, lse, tokens, accepted in runs:
            assert torch.equal(out[lo:hi], want[i][0][lo:hi]) and torch.equal(lse[lo:hi], want[i][1][lo:hi])
            assert torch.equal(tokens, drawn.tokens) and torch.equal(accepted, drawn.accepted)


@pytest.mark.parametrize("dtype,kv", KINDS)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("Hq,Hk,n,length", [(32, 32, 400, 250), (32, 8, 100, 60), (28, 4, 300, 275), (7, 7, 900, 700)])
def test_first_halves_of_tiles_that_see_no_key(dtype, kv, D, Hq, Hk, n, length):
    """More new tokens than cached ones, so that the first 128 rows of a tile see no key and the next 128 do, head
    behind head in one block: the same bits every time, and right."""
    att, s = check([n] * 4, [length - n] * 4, Hq, Hk, D, 16, dtype, kv, seed=n)
    want = call(att, s, return_lse=True)
    for _ in range(20):
        for a, b in zip(call(att, s, return_lse=True), want):
            assert torch.equal(a, b)


def bounded(att, s, out, lse, tries):
    """``ecah_paged_prefill_bounded``, enqueued."""
    ptr = lambda t: None if t is None else t.data_ptr()   # noqa: E731
    q, k, v = s["q"], s["k"], s["v"]
    half = 0 if q.dtype == torch.float16 else 1
    a = _abi.PrefillArgs(abi_version=_abi.ABI_VERSION, dtype=half, tokens=q.shape[0], num_qo_heads=q.shape[1], sm_scale=q.shape[2] ** -0.5,
                         causal=1, q=ptr(q), q_token_stride=q.stride(0), q_head_stride=q.stride(1), out=ptr(out),
                         out_token_stride=out.stride(0), out_head_stride=out.stride(1), lse=ptr(lse), qo_indptr=ptr(s["qo_indptr"]),
                         kv_last_page_len=ptr(s["last"]), workspace=ptr(att.prefill_workspace), workspace_bytes=att.prefill_workspace.numel())
    a.cache = _abi.KVCache(kv_dtype=_abi.KV_E4M3 if k.dtype == E4M3 else half, num_pages=k.shape[0], page_size=k.shape[1],
                           num_kv_heads=k.shape[2], head_dim=k.shape[3], batch=len(s["lengths"]), k_cache=ptr(k), v_cache=ptr(v),
                           k_page_stride=k.stride(0), k_slot_stride=k.stride(1), k_head_stride=k.stride(2), v_page_stride=v.stride(0),
                           v_slot_stride=v.stride(1), v_head_stride=v.stride(2), k_scale=ptr(s["ks"]), v_scale=ptr(s["vs"]),
                           kv_indptr=ptr(s["indptr"]), kv_indices=ptr(s["indices"]), num_indices=s["indices"].numel())
    assert _abi.lib().ecah_paged_prefill_bounded(ctypes.byref(a), tries, torch.cuda.current_stream().cuda_stream) == 0


@pytest.mark.parametrize("dtype,kv", KINDS)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_waits_of_a_few_tries_end_and_leave_the_next_launch_right(dtype, kv, D):
    """Limits that run out in the middle, with tiles under way by the copy engine: the launch ends, writes no row
    that is not the requests', and what follows on the same SMs and workspace is right."""
    s = setup([300, 5, 40], [0, 6000, 2000], 8, 2, D, 16, dtype, kv, behind=3, seed=23)
    att = PagedAttention(8, 2, D, 16, dtype, kv_dtype=kv, max_batch=3)
    T, hi = s["q"].shape[0], s["ptr"][-1]
    out, lse = torch.empty((T, 8, D), dtype=dtype, device=DEV), torch.empty((T, 8), device=DEV)
    for tries in (1, 2, 3, 5, 9, 30, 100):
        for limit in (tries, tries, 1 << 20):
            out.fill_(7.0); lse.fill_(7.0)
            bounded(att, s, out, lse, limit)
            torch.cuda.synchronize()
            assert bool((out[hi:] == 7.0).all()) and bool((lse[hi:] == 7.0).all())
        compare(s, out, lse)


@pytest.mark.parametrize("dtype,kv", KINDS)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_waits_that_run_out_for_some_give_nan_or_the_row(dtype, kv, D):
    """Some warps of a block give up while others go on: no row may hold products of what was not there yet.  Both
    many items of one tile of keys and few items of many."""
    for new, ctx in (([300, 5, 40], [0, 6000, 2000]), ([257] * 24, [0] * 24), ([900], [3000])):
        s = setup(new, ctx, 8, 2, D, 16, dtype, kv, seed=24)
        att = PagedAttention(8, 2, D, 16, dtype, kv_dtype=kv, max_batch=len(new))
        want, wlse, tol, ltol = reference(s["q"], s["ptr"], s["lengths"], s["indptr"], s["indices"], s["k"], s["v"], s["ks"], s["vs"],
                                          D ** -0.5, True)
        out, lse = torch.empty(want.shape, dtype=dtype, device=DEV), torch.empty(wlse.shape, device=DEV)
        for tries in (1, 1, 2, 2, 3, 4, 6, 10, 20, 50):
            out.fill_(7.0); lse.fill_(7.0)
            bounded(att, s, out, lse, tries)
            torch.cuda.synchronize()
            lost = torch.isnan(lse)
            assert bool(((out.double() - want).abs() <= tol)[~lost].all()) and bool(((lse.double() - wlse).abs() <= ltol)[~lost].all())
            assert bool(torch.isnan(out).all(-1)[lost].all())


def test_the_workspace_is_made_by_the_first_prefill(monkeypatch):
    """A handle that only decodes holds none; a capture cannot make it; handles and captures after that share nothing."""
    s = setup([40, 9], [3, 700], 8, 2, 128, 16, torch.float16, seed=25)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    att = PagedAttention(8, 2, 128, 16, torch.float16, max_batch=2)
    dec = att.decode(s["q"][:2], s["indptr"], s["indices"], s["last"], s["k"], s["v"])
    assert torch.cuda.memory_allocated() - before - att.workspace.numel() < 1 << 20
    assert torch.isfinite(dec).all()
    with monkeypatch.context() as m:
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        with pytest.raises(RuntimeError, match="inside a CUDA-graph capture"):
            call(att, s)
    assert att._prefill_workspace is None
    out, lse = call(att, s, return_lse=True)
    compare(s, out, lse)
    ws = att.prefill_workspace
    assert ws.numel() == paged.prefill_workspace_bytes(128) and att.prefill_workspace is ws
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, l2 = call(att, s, return_lse=True)
    graph.replay()
    assert torch.equal(got, out) and torch.equal(l2, lse)
    other = PagedAttention(8, 2, 128, 16, torch.float16, max_batch=2)
    assert other.prefill_workspace.data_ptr() != ws.data_ptr()       # reading it makes it


def with_scores(new, ctx, D, dtype, kv, at, score):
    """A batch of one request whose keys score 0, but key ``at`` as it says (scaled by 1); values random."""
    s = setup([new], [ctx], 4, 2, D, 16, dtype, kv, seed=26)
    q = torch.zeros_like(s["q"])
    q[..., 0] = 1.0
    s["q"] = q
    pg = s["indices"].long()
    (s["k"].view(torch.uint8) if kv else s["k"])[pg] = 0
    where = (pg[at // 16], slice(None), at % 16) if kv else (pg[at // 16], at % 16)
    if kv:
        s["k"].view(torch.uint8)[pg[at // 16], at % 16, :, 0] = torch.tensor(1.0 if score > 0 or score != score else -1.0).to(E4M3).view(torch.uint8).item()
        s["ks"][pg] = 1.0
        s["ks"][where] = abs(score)
    else:
        s["k"][where + (slice(None), 0)] = score
    return s


@pytest.mark.parametrize("dtype,kv", KINDS)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("score", [math.inf, math.nan, -math.inf])
def test_infinite_scores_reach_the_rows_that_see_them_alone(dtype, kv, D, score):
    """+inf and NaN: rows and log-sum-exp are NaN, in whole items and in ones joined of parts; -inf: no weight."""
    att = PagedAttention(4, 2, D, 16, dtype, kv_dtype=kv, max_batch=1)
    for new, ctx, at in ((200, 0, 150), (3, 9000, 40), (3, 9000, 8990), (300, 2000, 2100)):
        s = with_scores(new, ctx, D, dtype, kv, at, score)
        out, lse = call(att, s, return_lse=True, sm_scale=1.0)
        sees = torch.arange(ctx, ctx + new, device=DEV) >= at
        n = torch.arange(ctx + 1, ctx + new + 1, device=DEV).double()
        if score == -math.inf:
            n = n - sees.double()
            sees = torch.zeros_like(sees)
        assert torch.isnan(out[sees]).all() and torch.isnan(lse[sees]).all()
        assert torch.isfinite(out[~sees]).all()
        assert ((lse[~sees].double() - n[~sees].log()[:, None]).abs() <= 2e-5 + 4e-6 * 10).all()
        if new == 3:                              # decode: the same rules for the last token
            o, l = att.decode(s["q"][-1:], s["indptr"], s["indices"], s["last"], s["k"], s["v"], k_scale=s["ks"], v_scale=s["vs"],
                              sm_scale=1.0, return_lse=True)
            if score == -math.inf:
                assert torch.isfinite(o).all() and ((l.double() - n[-1].log()).abs() <= 6e-5).all()
            else:
                assert torch.isnan(o).all() and torch.isnan(l).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_a_row_of_scores_without_mass(dtype, D):
    """Every score -inf: zeros, and a log-sum-exp of -inf, in prefill and decode."""
    s = setup([70], [200], 4, 2, D, 16, dtype, seed=27)
    q = torch.zeros_like(s["q"])
    q[..., 0] = 1.0
    s["q"] = q
    pg = s["indices"].long()
    s["k"][pg] = 0.0
    s["k"][pg, :, :, 0] = -math.inf
    att = PagedAttention(4, 2, D, 16, dtype, max_batch=1)
    for out, lse in (call(att, s, return_lse=True), att.decode(q[:1], s["indptr"], s["indices"], s["last"], s["k"], s["v"], return_lse=True)):
        assert bool((out == 0).all()) and bool(torch.isneginf(lse).all())
