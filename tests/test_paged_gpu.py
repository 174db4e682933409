"""The paged append and the paged decode attention on the GPU against their
formulas in float64.

Tolerances, from the arithmetic (u = half a unit in the last place of the
output type, relative: 2^-8 for bf16 with its 7 stored bits, 2^-11 for f16 with
its 10):
  append: one rounding of a float32 result whose own error is a few 2^-23 of
    the row's largest magnitude: u |y| + 2^-18 max|y| (+ f16's subnormal step).
    e4m3: half a unit, 2^-4 |y| + 2^-10 scale, plus the same.
  decode: each softmax weight is rounded to the operand type (u of itself, and
    for f16 2^-25 of the row's largest), so |error| <= u |o| + u sum p|v| +
    2^-24 max(p) sum|v| + float32's 2^-16 sum p|v|.
"""
import ctypes
import math

import pytest
import torch

from ecahlang_b200 import _abi, paged
from ecahlang_b200.paged import PagedAttention

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3 = torch.float8_e4m3fn
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def pages_for(lengths, page, g, spare=3):
    counts = [-(-n // page) for n in lengths]
    total = sum(counts)
    order = torch.randperm(total + spare, generator=g, device=DEV)[:total].to(torch.int32)
    indptr = torch.tensor([0] + counts).cumsum(0).to(torch.int32).to(DEV)
    last = torch.tensor([(n - 1) % page + 1 if n else 0 for n in lengths], dtype=torch.int32, device=DEV)
    return total + spare, indptr, order, last


def cache_of(pages, page, heads, D, dtype, g, layout="nhd", fill="rand"):
    """k, v, k_scale, v_scale with NaN everywhere (fill='nan') or random."""
    shape = (pages, page, heads, D)
    if layout == "hnd":
        mk = lambda t: torch.empty((pages, heads, page, D), dtype=dtype, device=DEV).transpose(1, 2)   # noqa: E731
    elif layout == "paired":                     # [pages, 2, page, heads, D], one buffer
        both = torch.empty((pages, 2, page, heads, D), dtype=dtype, device=DEV)
        mk = lambda t: both[:, t]                                                                       # noqa: E731
    else:
        mk = lambda t: torch.empty(shape, dtype=dtype, device=DEV)                                      # noqa: E731
    k, v = mk(0), mk(1)
    scales = [None, None]
    if dtype == E4M3:
        scales = [torch.rand((pages, heads, page), generator=g, device=DEV) * 0.02 + 1e-3 for _ in range(2)]
    for t in (k, v):
        x = torch.randn(shape, generator=g, device=DEV)
        if dtype == E4M3:
            x = (x * 100).clamp(-448, 448)
        if fill == "nan":
            x.fill_(float("nan"))
        t.copy_(x.to(dtype))
    return k, v, *scales


def values(c, scale):
    x = c.float().double()
    return x if scale is None else x * scale.double().transpose(1, 2)[..., None]


def decode_reference(q, lengths, indptr, indices, k, v, ks, vs, sm_scale):
    B, Hq, D = q.shape
    Hk, page = k.shape[2], k.shape[1]
    out, tol = torch.zeros(B, Hq, D, dtype=torch.float64, device=DEV), torch.zeros(B, Hq, D, dtype=torch.float64, device=DEV)
    lse = torch.full((B, Hq), -math.inf, dtype=torch.float64, device=DEV)
    smax = torch.zeros(B, Hq, dtype=torch.float64, device=DEV)
    u = HALF[q.dtype]
    ptr = indptr.tolist()
    for b, n in enumerate(lengths):
        if not n:
            continue
        pg = indices[ptr[b]:ptr[b + 1]].long()
        sel = lambda c: (c.view(torch.uint8)[pg].view(E4M3) if c.dtype == E4M3 else c[pg])   # noqa: E731
        kk, vv = (values(sel(c), None if s is None else s[pg]).reshape(-1, Hk, D)[:n] for c, s in ((k, ks), (v, vs)))
        s = torch.einsum("hgd,nhd->hgn", q[b].double().view(Hk, Hq // Hk, D), kk) * sm_scale
        p = torch.softmax(s, -1)
        out[b] = torch.einsum("hgn,nhd->hgd", p, vv).reshape(Hq, D)
        mass = torch.einsum("hgn,nhd->hgd", p, vv.abs()).reshape(Hq, D)
        heavy = (p.amax(-1)[..., None] * vv.abs().sum(0)[:, None]).reshape(Hq, D)
        if vs is not None:   # weights carry the value's scale: the largest of p * scale, of the codes' sum
            w = torch.einsum("hgn,nh->hgn", p, vs[pg].double().transpose(1, 2).reshape(-1, Hk)[:n]).amax(-1)
            codes = sel(v).float().double().reshape(-1, Hk, D)[:n].abs().sum(0)
            heavy = (w[..., None] * codes[:, None]).reshape(Hq, D)
        tol[b] = u * out[b].abs() + (u + 2.0 ** -16) * mass + 2.0 ** -24 * heavy + 1e-7
        lse[b] = torch.logsumexp(s, -1).reshape(Hq)
        smax[b] = s.abs().amax(-1).reshape(Hq)
    return out, lse, tol, 2e-5 + 4e-6 * smax


def check_decode(lengths, Hq, Hk, D, page, dtype, kv=None, layout="nhd", seed=0, scale=1.5, sm_scale=None, listed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    pages, indptr, indices, last = pages_for(lengths, page, g)
    if listed:                               # a page list with room for more, as a captured step keeps it
        indices = torch.cat([indices, torch.full((listed,), -1, dtype=torch.int32, device=DEV)])
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
    B = len(lengths)
    q = (torch.randn(B, Hq + 3, D, generator=g, device=DEV) * scale).to(dtype)[:, 1:Hq + 1]   # strided
    att = PagedAttention(Hq, Hk, D, page, dtype, kv_dtype=kv, max_batch=B)
    out, lse = att.decode(q, indptr, indices, last, k, v, k_scale=ks, v_scale=vs, return_lse=True, sm_scale=sm_scale)
    want, wlse, tol, ltol = decode_reference(q, lengths, indptr, indices, k, v, ks, vs, sm_scale or 1 / math.sqrt(D))
    err = (out.double() - want).abs()
    assert torch.isfinite(out).all()
    assert (err <= tol).all(), float((err / tol).max())
    empty = torch.isinf(wlse)
    assert torch.equal(torch.isinf(lse), empty)
    assert ((lse.double() - wlse).abs()[~empty] <= ltol[~empty]).all()
    again, _ = att.decode(q, indptr, indices, last, k, v, k_scale=ks, v_scale=vs, return_lse=True, sm_scale=sm_scale)
    assert torch.equal(out, again)
    return att


KINDS = [(torch.float16, None), (torch.bfloat16, None), (torch.float16, E4M3), (torch.bfloat16, E4M3)]


@pytest.mark.parametrize("dtype,kv", KINDS)
@pytest.mark.parametrize("D", [64, 96, 128, 192, 256])
def test_decode_head_dims(dtype, kv, D):
    check_decode([1, 0, 15, 16, 17, 63, 64, 65, 700, 0, 1900], 8, 2, D, 16, dtype, kv, seed=D)


@pytest.mark.parametrize("dtype,kv", KINDS)
@pytest.mark.parametrize("Hq,Hk", [(1, 1), (7, 1), (8, 8), (16, 2), (14, 2), (16, 1), (17, 1), (40, 2), (71, 1)])
def test_decode_groups(dtype, kv, Hq, Hk):
    check_decode([1, 130, 33, 1025], Hq, Hk, 128, 16, dtype, kv, seed=Hq)


@pytest.mark.parametrize("dtype,kv", KINDS)
@pytest.mark.parametrize("page", [1, 2, 5, 16, 64, 100, 1000])
@pytest.mark.parametrize("layout", ["nhd", "hnd", "paired"])
def test_decode_pages_and_layouts(dtype, kv, page, layout):
    check_decode([3, 999, 1000, 1001, 0, 128], 16, 4, 64, page, dtype, kv, layout, seed=page)


@pytest.mark.parametrize("dtype,kv", KINDS)
@pytest.mark.parametrize("lengths", [[1], [0], [0, 0, 0], [40000], [5, 70001, 1], [1] * 300, [513] * 37, [7] * 148 + [9000]])
def test_decode_lengths(dtype, kv, lengths):
    """Alone and long (joined over many blocks), many and short (several to a block)."""
    check_decode(lengths, 16, 2, 128, 16, dtype, kv, seed=len(lengths))


@pytest.mark.parametrize("dtype,kv", KINDS)
@pytest.mark.parametrize("scale,sm_scale", [(0.0, None), (40.0, None), (1.0, 3.0), (1e-3, 1e-3)])
def test_decode_score_ranges(dtype, kv, scale, sm_scale):
    """All weights alike, and one key that takes nearly all of it."""
    check_decode([300, 2000, 1], 8, 2, 128, 16, dtype, kv, scale=scale, sm_scale=sm_scale)


@pytest.mark.parametrize("dtype,kv", KINDS)
@pytest.mark.parametrize("Hq,Hk,D", [(16, 2, 128), (32, 8, 128), (32, 8, 64), (12, 6, 96), (8, 4, 256), (32, 4, 192),
                                     (64, 4, 128), (5, 5, 64), (40, 2, 64), (34, 2, 256), (7, 1, 192)])
@pytest.mark.parametrize("page", [5, 16])
def test_decode_with_a_long_page_list(dtype, kv, Hq, Hk, D, page):
    """The kernels of much work: chosen by the pages listed, whatever the lengths are."""
    check_decode([1, 0, 15, 16, 17, 63, 64, 65, 700, 0, 1900, 5000, 129], Hq, Hk, D, page, dtype, kv, seed=D + Hq,
                 listed=2_000_000 // (page * Hk))


@pytest.mark.parametrize("dtype,kv", KINDS)
def test_decode_much_work(dtype, kv):
    check_decode([40001, 0, 1, 39000, 77, 3001], 32, 8, 128, 16, dtype, kv)


@pytest.mark.parametrize("kv", [None, E4M3])
def test_decode_nan_and_infinite_keys_stay_in_their_row(kv):
    g = torch.Generator(device=DEV).manual_seed(1)
    pages, indptr, indices, last = pages_for([300, 300, 300], 16, g)
    k, v, ks, vs = cache_of(pages, 16, 2, 128, kv or torch.bfloat16, g)
    q = torch.randn(3, 8, 128, generator=g, device=DEV).bfloat16()
    att = PagedAttention(8, 2, 128, 16, torch.bfloat16, kv_dtype=kv)
    clean = att.decode(q, indptr, indices, last, k, v, k_scale=ks, v_scale=vs)
    page = int(indices[int(indptr[1]) + 3])
    if kv is None:
        k[page, 5, 0, 7] = float("nan")
        v[page, 6, 1, 9] = float("nan")
    else:
        ks[page, 0, 5] = float("nan")
        vs[page, 1, 6] = float("nan")
    got = att.decode(q, indptr, indices, last, k, v, k_scale=ks, v_scale=vs)
    assert torch.equal(got[[0, 2]], clean[[0, 2]])
    assert torch.isnan(got[1, :4]).all()
    assert torch.isnan(got[1, 4:, 9]).all()
    assert torch.isfinite(got[1, 4:]).any() == (kv is None)


def test_decode_offsets_past_32_bits():
    D, Hk, page = 128, 8, 16
    pages = (1 << 31) // (D * Hk * page) + 64
    k = torch.empty(pages, page, Hk, D, dtype=torch.float16, device=DEV)
    v = torch.empty_like(k)
    g = torch.Generator(device=DEV).manual_seed(2)
    indices = torch.tensor([pages - 1, 0, pages - 2, 1, pages - 7], dtype=torch.int32, device=DEV)
    small = torch.randn(2, 5, page, Hk, D, generator=g, device=DEV).half()
    k[indices.long()], v[indices.long()] = small[0], small[1]
    indptr = torch.tensor([0, 5], dtype=torch.int32, device=DEV)
    last = torch.tensor([9], dtype=torch.int32, device=DEV)
    q = torch.randn(1, 16, D, generator=g, device=DEV).half()
    att = PagedAttention(16, Hk, D, page, torch.float16)
    out = att.decode(q, indptr, indices, last, k, v)
    near = att.decode(q, indptr, torch.arange(5, dtype=torch.int32, device=DEV), last, small[0], small[1])
    assert torch.equal(out, near)
    new = torch.randn(2, Hk, D, generator=g, device=DEV).half()
    pos = torch.tensor([4 * page + 9, 9], dtype=torch.int32, device=DEV)
    att.append(None, new, new, pos, torch.zeros(2, dtype=torch.int32, device=DEV), indptr, indices, k, v)
    assert torch.equal(k[pages - 7, 9], new[0]) and torch.equal(v[pages - 1, 9], new[1])


def test_decode_many_shapes_on_one_workspace_streams_and_graph():
    g = torch.Generator(device=DEV).manual_seed(5)
    att = PagedAttention(16, 2, 128, 16, torch.bfloat16, max_batch=64)
    k, v, _, _ = cache_of(700, 16, 2, 128, torch.bfloat16, g)
    for lengths in ([9000], [17] * 64, [1], [3000, 0, 1], [9000]):
        _, indptr, indices, last = pages_for(lengths, 16, g)
        q = torch.randn(len(lengths), 16, 128, generator=g, device=DEV).bfloat16()
        want, _, tol, _ = decode_reference(q, lengths, indptr, indices, k, v, None, None, 128 ** -0.5)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            out = att.decode(q, indptr, indices, last, k, v)
        torch.cuda.current_stream().wait_stream(side)
        assert ((out.double() - want).abs() <= tol).all()
    # one captured launch, replayed with other lengths (a bucket of a captured decode step)
    lengths = [700, 20, 0, 1500]
    _, indptr, indices, last = pages_for([1600] * 4, 16, g)
    q = torch.randn(4, 16, 128, generator=g, device=DEV).bfloat16()
    ip, ix, la, out = torch.zeros_like(indptr), torch.zeros_like(indices), torch.zeros_like(last), torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        att.decode(q, ip, ix, la, k, v, out=out)
    for n in (lengths, [1, 0, 0, 0], [1600] * 4):
        _, indptr, indices, last = pages_for(n, 16, g)
        ip.copy_(indptr)
        ix[:len(indices)] = indices
        la.copy_(last)
        graph.replay()
        want, _, tol, _ = decode_reference(q, n, indptr, indices, k, v, None, None, 128 ** -0.5)
        assert ((out.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("Hq,Hk,D", [(32, 8, 128), (64, 4, 128), (8, 8, 192), (32, 2, 192)])
def test_decode_wait_that_runs_out_gives_nan_in_every_row(dtype, Hq, Hk, D):
    """With no tries for the copy engine's waits (its copies still land) nothing finite is left of a
    request with tokens; the launch after it finds its workspace as it should be."""
    g = torch.Generator(device=DEV).manual_seed(9)
    lengths = [20000, 0, 3, 700, 64]
    pages, indptr, indices, last = pages_for(lengths, 16, g)
    indices = torch.cat([indices, torch.full((2_000_000 // (16 * Hk),), -1, dtype=torch.int32, device=DEV)])
    k, v, _, _ = cache_of(pages, 16, Hk, D, dtype, g)
    q = torch.randn(len(lengths), Hq, D, generator=g, device=DEV).to(dtype)
    att = PagedAttention(Hq, Hk, D, 16, dtype, max_batch=len(lengths))
    out, lse = torch.zeros_like(q), torch.zeros(len(lengths), Hq, device=DEV)
    page, slot, head, _ = k.stride()
    cache = _abi.KVCache(kv_dtype=paged._DTYPES[dtype], num_pages=pages, page_size=16, num_kv_heads=Hk, head_dim=D,
                         batch=len(lengths), k_cache=k.data_ptr(), v_cache=v.data_ptr(), k_page_stride=page,
                         k_slot_stride=slot, k_head_stride=head, v_page_stride=page, v_slot_stride=slot,
                         v_head_stride=head, kv_indptr=indptr.data_ptr(), kv_indices=indices.data_ptr(),
                         num_indices=indices.numel())
    a = _abi.DecodeArgs(abi_version=_abi.ABI_VERSION, dtype=paged._DTYPES[dtype], num_qo_heads=Hq, sm_scale=D ** -0.5,
                        q=q.data_ptr(), q_token_stride=Hq * D, q_head_stride=D, out=out.data_ptr(),
                        out_token_stride=Hq * D, out_head_stride=D, lse=lse.data_ptr(),
                        kv_last_page_len=last.data_ptr(), cache=cache, workspace=att.workspace.data_ptr(),
                        workspace_bytes=att.workspace.numel())
    stream = torch.cuda.current_stream().cuda_stream
    assert _abi.lib().ecah_paged_decode_bounded(ctypes.byref(a), 0, stream) == 0
    some = torch.tensor(lengths, device=DEV) > 0
    assert torch.isnan(out[some]).all() and torch.isnan(lse[some]).all()
    assert (out[~some] == 0).all() and (lse[~some] == -math.inf).all()
    assert _abi.lib().ecah_paged_decode_bounded(ctypes.byref(a), 1 << 20, stream) == 0
    want, wlse = att.decode(q, indptr, indices, last, k, v, return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, wlse) and torch.isfinite(want).all()


# ------------------------------------------------------------------- append
def turn(x, w, eps, table, pos, interleaved):
    x = x.double()
    if w is not None:
        x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps) * w.double()
    if table is None:
        return x
    D = x.shape[-1]
    cs = table.double()[pos.long().clamp(0, table.shape[0] - 1)][:, None]
    c, s = cs[..., :D // 2], cs[..., D // 2:]
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :D // 2], x[..., D // 2:])
    y = torch.empty_like(x)
    if interleaved:
        y[..., 0::2], y[..., 1::2] = a * c - b * s, b * c + a * s
    else:
        y[..., :D // 2], y[..., D // 2:] = a * c - b * s, b * c + a * s
    return y


def table_of(rows, D):
    ang = torch.arange(rows, dtype=torch.float64)[:, None] * 1e6 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    return torch.cat([ang.cos(), ang.sin()], 1).float().to(DEV)


@pytest.mark.parametrize("dtype,kv", KINDS)
@pytest.mark.parametrize("D,Hq,Hk,T,page,layout,norm,rope,interleaved", [
    (128, 16, 2, 1, 16, "nhd", False, True, False),
    (128, 32, 8, 129, 16, "nhd", True, True, False),
    (64, 14, 2, 77, 5, "hnd", False, True, True),
    (96, 7, 1, 33, 1, "paired", True, True, True),
    (192, 4, 4, 50, 64, "nhd", True, False, False),
    (256, 8, 1, 300, 16, "hnd", True, True, False),
    (128, 5, 5, 9, 16, "nhd", False, False, False),
    (96, 6, 2, 40, 16, "nhd", True, True, False),
    (192, 8, 2, 21, 16, "paired", False, True, True),
])
def test_append(dtype, kv, D, Hq, Hk, T, page, layout, norm, rope, interleaved):
    g = torch.Generator(device=DEV).manual_seed(D + T)
    lengths = [60, 1 + T, 40]
    pages, indptr, indices, _ = pages_for(lengths, page, g)
    k, v, ks, vs = cache_of(pages, page, Hk, D, kv or dtype, g, layout)
    before = [None if t is None else t.clone() for t in (k, v, ks, vs)]
    qkv = (torch.randn(T, Hq + 2 * Hk, D, generator=g, device=DEV) * 2).to(dtype)
    qkv[T // 2, Hq] = 0                                # a key of zeros
    q, kn, vn = qkv.split([Hq, Hk, Hk], 1)
    batch = torch.ones(T, dtype=torch.int32, device=DEV)
    pos = torch.arange(1, T + 1, dtype=torch.int32, device=DEV)
    if T > 8:                                          # tokens of another request, and some that go nowhere
        batch[3], pos[3] = 2, 39
        batch[4] = -1
        batch[5] = 3
        pos[6] = (-(-lengths[1] // page)) * page       # past the request's pages
        pos[7] = -1
    wq, wk = ((torch.rand(D, generator=g, device=DEV) + 0.5).to(dtype) for _ in range(2)) if norm else (None, None)
    table = table_of(max(lengths) - 5, D) if rope else None
    att = PagedAttention(Hq, Hk, D, page, dtype, kv_dtype=kv)
    got = att.append(q, kn, vn, pos, batch, indptr, indices, k, v, k_scale=ks, v_scale=vs, cos_sin=table, q_norm=wq,
                     k_norm=wk, eps=1e-5, interleaved=interleaved)
    u = HALF[dtype]

    def near(y, want):
        big = want.abs().amax(-1, keepdim=True)
        assert ((y.double() - want).abs() <= u * want.abs() + 2.0 ** -18 * big + 2.0 ** -25).all()

    near(got, turn(q, wq, 1e-5, table, pos, interleaved))
    written = torch.zeros(pages, page, dtype=torch.bool, device=DEV)
    rows = [t for t in range(T) if not (T > 8 and t in (4, 5, 6, 7))]
    ptr, ind = indptr.tolist(), indices.tolist()
    at = torch.tensor([[ind[ptr[int(batch[t])] + int(pos[t]) // page], int(pos[t]) % page] for t in rows], device=DEV)
    written[at[:, 0], at[:, 1]] = True
    for c, sc, new, old, osc in ((k, ks, turn(kn, wk, 1e-5, table, pos, interleaved), before[0], before[2]),
                                 (v, vs, vn.double(), before[1], before[3])):
        new = new[rows]
        if kv is None:
            near(c[at[:, 0], at[:, 1]], new)
        else:
            s = sc[at[:, 0], :, at[:, 1]].double()
            torch.testing.assert_close(s, new.abs().amax(-1).clamp_min(448e-12) / 448, rtol=1e-5, atol=0)
            code = c.view(torch.uint8)[at[:, 0], at[:, 1]].view(E4M3).float().double()
            err = (code * s[..., None] - new).abs()
            assert (err <= 2.0 ** -4 * new.abs() + 2.0 ** -10 * s[..., None] + 2.0 ** -18 * new.abs().amax(-1, keepdim=True)).all()
            assert torch.equal(sc.transpose(1, 2)[~written], osc.transpose(1, 2)[~written])
        raw = [t.contiguous().view(torch.uint8 if kv else torch.int16) for t in (c, old)]
        assert torch.equal(raw[0][~written], raw[1][~written])


@pytest.mark.parametrize("kv", [None, E4M3])
def test_append_in_place_and_without_queries(kv):
    g = torch.Generator(device=DEV).manual_seed(4)
    pages, indptr, indices, _ = pages_for([64], 16, g)
    att = PagedAttention(8, 2, 128, 16, torch.float16, kv_dtype=kv)
    a, b, c = (att.new_cache(pages) for _ in range(3))
    qkv = torch.randn(40, 12, 128, generator=g, device=DEV).half()
    pos, batch = torch.arange(40, dtype=torch.int32, device=DEV), torch.zeros(40, dtype=torch.int32, device=DEV)
    table = table_of(64, 128)
    q, k, v = qkv.split([8, 2, 2], 1)
    want = att.append(q, k, v, pos, batch, indptr, indices, a[0], a[1], k_scale=a[2], v_scale=a[3], cos_sin=table)
    att.append(None, k, v, pos, batch, indptr, indices, b[0], b[1], k_scale=b[2], v_scale=b[3], cos_sin=table)
    got = att.append(q, k, v, pos, batch, indptr, indices, c[0], c[1], k_scale=c[2], v_scale=c[3], cos_sin=table, q_out=q)
    assert got.data_ptr() == q.data_ptr() and torch.equal(got, want)
    for other in (b, c):
        for x, y in zip(a, other):
            assert x is None or torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_append_nan_inf_and_tiny_rows_e4m3():
    g = torch.Generator(device=DEV).manual_seed(4)
    att = PagedAttention(1, 1, 64, 16, torch.bfloat16, kv_dtype=E4M3)
    k, v, ks, vs = att.new_cache(1)
    x = torch.randn(5, 1, 64, generator=g, device=DEV).bfloat16()
    x[1, 0, 3] = float("nan")
    x[2, 0, 3] = float("inf")
    x[3] = 1e-20
    x[4] = 1e30
    ip, ix = torch.tensor([0, 1], dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    att.append(None, x, x, torch.arange(5, dtype=torch.int32, device=DEV), torch.zeros(5, dtype=torch.int32, device=DEV),
               ip, ix, k, v, k_scale=ks, v_scale=vs)
    got = k[0, :5, 0].float() * ks[0, 0, :5, None]
    assert torch.isfinite(got[[0, 3, 4]]).all()
    assert torch.isnan(got[1]).all() and not torch.isfinite(got[2]).any()
    assert (got[3].abs() <= 1e-14).all()
    torch.testing.assert_close(got[4], x[4, 0].float(), rtol=2 ** -4, atol=0)


def test_step_appends_then_decodes():
    """Tokens appended one by one give the attention over all of them."""
    g = torch.Generator(device=DEV).manual_seed(6)
    for kv in (None, E4M3):
        att = PagedAttention(8, 2, 64, 16, torch.float16, kv_dtype=kv, max_batch=2)
        cache = att.new_cache(8)
        indptr = torch.tensor([0, 2, 4], dtype=torch.int32, device=DEV)
        indices = torch.tensor([5, 1, 7, 0], dtype=torch.int32, device=DEV)
        table = table_of(32, 64)
        batch = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
        for step in range(20):
            qkv = torch.randn(2, 12, 64, generator=g, device=DEV).half()
            q, k, v = qkv.split([8, 2, 2], 1)
            pos = torch.full((2,), step, dtype=torch.int32, device=DEV)
            n = step // 16 + 1
            ip = torch.tensor([0, n, 2 * n], dtype=torch.int32, device=DEV)
            ix = indices.view(2, 2)[:, :n].reshape(-1).contiguous()
            q = att.append(q, k, v, pos, batch, indptr, indices, cache[0], cache[1], k_scale=cache[2], v_scale=cache[3],
                           cos_sin=table)
            last = torch.full((2,), step % 16 + 1, dtype=torch.int32, device=DEV)
            out = att.decode(q, ip, ix, last, cache[0], cache[1], k_scale=cache[2], v_scale=cache[3])
            want, _, tol, _ = decode_reference(q, [step + 1] * 2, ip, ix, *cache, 1 / 8)
            assert ((out.double() - want).abs() <= tol).all()


def test_custom_ops():
    g = torch.Generator(device=DEV).manual_seed(7)
    att = PagedAttention(8, 2, 128, 16, torch.float16)
    pages, indptr, indices, last = pages_for([40, 3], 16, g)
    a, b = att.new_cache(pages), att.new_cache(pages)
    q, k, v = torch.randn(2, 12, 128, generator=g, device=DEV).half().split([8, 2, 2], 1)
    pos, batch = torch.tensor([39, 2], dtype=torch.int32, device=DEV), torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    want = att.append(q, k, v, pos, batch, indptr, indices, a[0], a[1], cos_sin=table_of(40, 128))
    qo = torch.empty(2, 8, 128, dtype=torch.float16, device=DEV)
    torch.ops.ecah.paged_append(q, k, v, pos, batch, indptr, indices, b[0], b[1], None, None, table_of(40, 128), None, None,
                                1e-6, False, qo)
    assert torch.equal(qo, want) and torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    out = torch.empty_like(qo)
    torch.ops.ecah.paged_decode(qo, indptr, indices, last, b[0], b[1], None, None, 128 ** -0.5, out, None, att.workspace)
    assert torch.equal(out, att.decode(want, indptr, indices, last, a[0], a[1]))


def test_bad_indices_are_clamped():
    """Index arrays with entries outside the cache read inside it."""
    g = torch.Generator(device=DEV).manual_seed(8)
    k, v, _, _ = cache_of(4, 16, 2, 64, torch.float16, g)
    q = torch.randn(3, 8, 64, generator=g, device=DEV).half()
    att = PagedAttention(8, 2, 64, 16, torch.float16)
    t = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)   # noqa: E731
    out = att.decode(q, t(0, 2, 3, 9), t(-7, 99, 1, 2), t(5, 99, -3), k, v)
    # pages 0 and 3 with 5 in the last; page 1 whole; the list cut at its end: pages 1 entry (2), none of its tokens
    want, _, tol, _ = decode_reference(q, [21, 16, 0], t(0, 2, 3, 4), t(0, 3, 1, 2), k, v, None, None, 1 / 8)
    assert ((out.double() - want).abs() <= tol).all()


def test_empty_and_refused():
    att = PagedAttention(8, 2, 64, 16, torch.float16, max_batch=4)
    k, v, _, _ = att.new_cache(3)
    t = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)   # noqa: E731
    z = lambda *s, d=torch.float16: torch.zeros(*s, dtype=d, device=DEV)   # noqa: E731
    assert att.decode(z(0, 8, 64), t(0), t(), t(), k, v).shape == (0, 8, 64)
    assert att.append(z(0, 8, 64), z(0, 2, 64), z(0, 2, 64), t(), t(), t(0), t(), k, v).shape == (0, 8, 64)
    none = PagedAttention(8, 2, 64, 16, torch.float16).new_cache(0)
    assert (att.decode(z(1, 8, 64) + 1, t(0, 1), t(0), t(5), none[0], none[1]) == 0).all()
    ok = dict(q=z(1, 8, 64), kv_indptr=t(0, 1), kv_indices=t(0), kv_last_page_len=t(3), k_cache=k, v_cache=v)
    paged.decode(**ok, workspace=att.workspace)
    for bad in (dict(q=z(1, 7, 64)), dict(q=z(2, 8, 64)), dict(q=z(1, 8, 64).float()), dict(q=z(1, 8, 128)),
                dict(kv_indptr=t(0, 1).long()), dict(kv_indices=t(0).cpu()), dict(kv_last_page_len=t(3, 3)),
                dict(v_cache=v[:2]), dict(k_cache=k.bfloat16()), dict(k_cache=k[..., :48], v_cache=v[..., :48]),
                dict(k_scale=z(3, 2, 16, d=torch.float32)), dict(sm_scale=0.0), dict(sm_scale=float("inf")),
                dict(out=z(1, 8, 63)), dict(lse=z(1, 7, d=torch.float32)), dict(workspace=att.workspace[:8]),
                dict(workspace=att.workspace.int()), dict(q=z(1, 8, 128)[..., ::2]), dict(kv_indptr=t()),
                dict(k_cache=k.view(torch.uint8).view(E4M3), v_cache=v.view(torch.uint8).view(E4M3))):
        with pytest.raises(RuntimeError):
            paged.decode(**{**ok, "workspace": att.workspace, **bad})
    with pytest.raises(RuntimeError, match="max_batch"):
        att.decode(z(5, 8, 64), t(0, 1, 1, 1, 1, 1), t(0), t(3, 0, 0, 0, 0), k, v)
    ok = dict(q=z(2, 8, 64), k=z(2, 2, 64), v=z(2, 2, 64), positions=t(0, 1), batch_index=t(0, 0), kv_indptr=t(0, 1),
              kv_indices=t(0), k_cache=k, v_cache=v)
    paged.append(**ok)
    for bad in (dict(k=z(2, 2, 64).float()), dict(v=z(2, 1, 64)), dict(v=z(2, 2, 64).bfloat16()), dict(q=z(3, 8, 64)),
                dict(positions=t(0)), dict(batch_index=t(0, 0).long()), dict(cos_sin=z(4, 64)),
                dict(cos_sin=z(0, 64, d=torch.float32)), dict(cos_sin=z(4, 32, d=torch.float32)), dict(q_norm=z(63)),
                dict(k_norm=z(64, d=torch.float32)), dict(q_out=z(2, 8, 64, d=torch.bfloat16)),
                dict(q=None, q_norm=z(64)), dict(k_scale=z(3, 2, 16, d=torch.float32)), dict(k=z(2, 2, 65)[..., 1:])):
        with pytest.raises(RuntimeError):
            paged.append(**{**ok, **bad})
    for bad in (dict(head_dim=80), dict(num_qo_heads=9), dict(page_size=0), dict(dtype=torch.float32),
                dict(kv_dtype=torch.bfloat16), dict(max_batch=0)):
        with pytest.raises(RuntimeError):
            PagedAttention(**{**dict(num_qo_heads=8, num_kv_heads=2, head_dim=64, page_size=16, dtype=torch.float16), **bad})
