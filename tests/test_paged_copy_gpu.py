"""Page copies on the GPU against indexing: bytes are equal, and nothing else is written."""
import pytest
import torch

from ecahlang_b200 import paged
from ecahlang_b200.paged import PagedAttention
from test_paged_gpu import E4M3, cache_of

pytestmark = pytest.mark.gpu
DEV = "cuda"


def raw(t):
    return t.view(torch.uint8) if t.dtype == E4M3 else t


def copied(caches, src, dst, tokens):
    """What the caches should hold, layer by layer."""
    out = []
    for k, v, ks, vs in caches:
        new = [raw(k).clone(), raw(v).clone(), None if ks is None else ks.clone(), None if vs is None else vs.clone()]
        for s, d, n in zip(src, dst, tokens):
            if s == d or not (0 <= s < k.shape[0] and 0 <= d < k.shape[0]):
                continue
            for i, t in enumerate((raw(k), raw(v))):
                new[i][d, :n] = t[s, :n]
            for i, t in ((2, ks), (3, vs)):
                if t is not None:
                    new[i][d, :, :n] = t[s, :, :n]
        out.append(new)
    return out


def check(caches, call, src, dst, tokens):
    want = copied(caches, src, dst, tokens)
    call()
    for got, new in zip(caches, want):
        for a, b in zip(got, new):
            assert (a is None) == (b is None)
            if a is not None:
                assert torch.equal(raw(a), b)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, E4M3])
@pytest.mark.parametrize("D", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("page,heads", [(1, 1), (16, 2), (7, 5), (64, 1)])
@pytest.mark.parametrize("layout", ["nhd", "hnd", "paired"])
def test_layouts(dtype, D, page, heads, layout):
    g = torch.Generator(device=DEV).manual_seed(D + page)
    caches = [cache_of(20, page, heads, D, dtype, g, layout) for _ in range(3)]
    src, dst = [3, 3, 0, 19, -1, 5, 6, 20, 8], [4, 1, 2, 18, 9, 5, -3, 10, 11]
    tokens = [page, 0, 1, max(1, page - 1), page, page, page, page, page // 2]
    t = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in (src, dst, tokens)]
    check(caches, lambda: paged.copy_pages(t[0], t[1], caches, tokens=t[2]), src, dst, tokens)
    check(caches, lambda: paged.copy_pages(t[0], t[1], caches), src, dst, [page] * len(src))


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
def test_strides_that_leave_gaps(dtype):
    """Slots and heads with room between them: neither is one run with its neighbour."""
    g = torch.Generator(device=DEV).manual_seed(1)
    kv = dtype
    big = [torch.zeros((9, 8, 4, 256), dtype=torch.uint8 if kv == E4M3 else kv, device=DEV).view(kv) for _ in range(2)]
    for b in big:
        raw(b).copy_(torch.randint(0, 255, b.shape, generator=g, device=DEV).to(raw(b).dtype))
    for cut in (lambda b: b[:, :, :3, :64], lambda b: b[:, :5, :, :], lambda b: b[:, 1:7:2, 1:2], lambda b: b[:, :, ::2, :128]):
        k, v = (cut(b) for b in big)
        s = [None, None] if kv != E4M3 else [torch.rand((9, k.shape[2], k.shape[1]), generator=g, device=DEV) for _ in range(2)]
        before = [raw(b).clone() for b in big]
        src, dst, tokens = [0, 1], [7, 3], [k.shape[1], 2]
        check([(k, v, *s)], lambda: paged.copy_pages(src, dst, [(k, v, *s)], tokens=tokens), src, dst, tokens)
        for b, old in zip(big, before):                      # nothing beside the cache
            now = raw(b).clone()
            cut(now).copy_(cut(old))
            assert torch.equal(now, old)


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
def test_no_tokens_of_pages_with_gaps(dtype):
    """Zero tokens and fewer copy nothing, also where a slot does not follow its neighbour."""
    g = torch.Generator(device=DEV).manual_seed(6)
    big = [torch.zeros((9, 8, 4, 256), dtype=torch.uint8 if dtype == E4M3 else dtype, device=DEV).view(dtype) for _ in range(2)]
    for b in big:
        raw(b).copy_(torch.randint(0, 255, b.shape, generator=g, device=DEV).to(raw(b).dtype))
    cuts = [lambda b: b[:, :, :3, :64], lambda b: b[:, :5, :, :], lambda b: b[:, 1:7:2, 1:2], lambda b: b[:, :, ::2, :128],
            lambda b: b[:, :, 1::2, 64:128]]
    for cut in cuts:
        k, v = (cut(b) for b in big)
        s = [None, None] if dtype != E4M3 else [torch.rand((9, k.shape[2], k.shape[1]), generator=g, device=DEV) for _ in range(2)]
        src, dst, tokens = [0, 1, 2, 4], [7, 3, 5, 8], [0, -3, 0, 2]
        t = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in (src, dst, tokens)]
        check([(k, v, *s)], lambda: paged.copy_pages(t[0], t[1], [(k, v, *s)], tokens=t[2]), src, dst, [max(n, 0) for n in tokens])


def test_many_layers_and_pairs():
    g = torch.Generator(device=DEV).manual_seed(2)
    att = PagedAttention(8, 2, 64, 16, torch.float16, kv_dtype=E4M3)
    caches = [cache_of(300, 16, 2, 64, E4M3, g) for _ in range(130)]
    order = torch.randperm(300, generator=g, device=DEV).tolist()
    src, dst = order[:150], order[150:]
    tokens = torch.randint(0, 17, (150,), generator=g, device=DEV).tolist()
    check(caches, lambda: att.copy_pages(src, dst, caches, tokens=tokens), src, dst, tokens)


def test_tokens_beyond_the_page_are_clamped():
    g = torch.Generator(device=DEV).manual_seed(3)
    caches = [cache_of(6, 16, 2, 64, torch.float16, g)]
    t = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([0, 1], [2, 3], [99, -5])]
    check(caches, lambda: paged.copy_pages(t[0], t[1], caches, tokens=t[2]), [0, 1], [2, 3], [16, 0])


def test_captured_and_replayed():
    g = torch.Generator(device=DEV).manual_seed(4)
    caches = [cache_of(40, 16, 2, 128, torch.bfloat16, g) for _ in range(2)]
    t = [torch.full((6,), -1, dtype=torch.int32, device=DEV) for _ in range(3)]
    paged.copy_pages(t[0], t[1], caches, tokens=t[2])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.copy_pages(t[0], t[1], caches, tokens=t[2])
    for src, dst, tokens in (([1, 2, -1, -1, -1, -1], [10, 11, -1, -1, -1, -1], [3, 16, 0, 0, 0, 0]),
                             ([9, 9, 9, 9, 9, 9], [20, 21, 22, 23, 24, 25], [1, 2, 3, 4, 5, 16])):
        for a, b in zip(t, (src, dst, tokens)):
            a.copy_(torch.tensor(b))
        check(caches, graph.replay, src, dst, tokens)


def test_refusals():
    g = torch.Generator(device=DEV).manual_seed(5)
    att = PagedAttention(8, 2, 64, 16, torch.float16)
    c, other = cache_of(6, 16, 2, 64, torch.float16, g), cache_of(6, 16, 2, 64, E4M3, g)
    i = torch.zeros(2, dtype=torch.int32, device=DEV)
    for caches, why in (([c, other], "must be|one shape"), ([cache_of(6, 16, 2, 64, torch.float32, g)], "unsupported cache dtype"),
                        ([(c[0], c[1][:5], None, None)], "must be"), ([c[:2]], "expected"), ([(c[0], c[1], other[2], other[3])], "no scales"),
                        ([(other[0], other[1], None, None)], "needs k_scale|must be"), ([c, cache_of(6, 16, 2, 64, torch.float16, g, "hnd")], "one shape"),
                        ([c, cache_of(7, 16, 2, 64, torch.float16, g)], "one shape"), ([cache_of(6, 8, 2, 64, torch.float16, g)], "must be"),
                        ([(c[0][:1].expand(6, 16, 2, 64), c[1], None, None)], "share memory")):
        with pytest.raises(RuntimeError, match=why):
            att.copy_pages(i, i, caches)
    for src, dst, tokens, why in ((i.long(), i, None, "src"), (i, i[:1], None, "dst"), (i, i, i[:1], "tokens"), (i, [1, 2], None, "all host"),
                                  ([0], [1], i[:1], "all host")):
        with pytest.raises(RuntimeError, match=why):
            att.copy_pages(src, dst, [c], tokens=tokens)
    e = [other, tuple(t.clone() for t in other)]
    want = copied(e, [0], [5], [16])
    torch.ops.ecah.paged_copy(i[:1], i[:1] + 5, None, [x[0] for x in e], [x[1] for x in e], [x[2] for x in e], [x[3] for x in e])
    assert all(torch.equal(raw(a), b) for x, w in zip(e, want) for a, b in zip(x, w))
