"""Long decode attention in float64, on any device: inputs under which a lost or
misweighted run of keys shows, and a tolerance that it exceeds.

Values follow waves over the key's place, so that the output is small beside
them and every run of keys moves some dimension of it.  The tolerance takes the
rounding of the softmax weights at its own size: a weight is off by at most u of
itself (u of the operand type: f16 for f16 and e4m3 caches, bf16 for bf16) with
a sign that the keys do not share, standard deviation at most u / sqrt(3), so
eight times u sqrt(sum p^2 v^2) is 13 deviations.  Beside it stand the output's
rounding u |o|, float32's part 2^-16 sum p |v| (scores of a magnitude up to 16
rounded a few times, exponentials, sums), and half of f16's smallest weight at
2^-32 of the largest (twice that, since e4m3 weights carry scales that differ by
a quarter).
"""
import math

import torch

E4M3 = torch.float8_e4m3fn
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}     # half a unit in the last place


def long_cache(n, page, heads, D, dtype, kv, gen, device):
    """k, v [pages, page, heads, D] and scales (None, or of an e4m3 cache) of one request of n tokens in page order."""
    pages = -(-n // page)
    shape = (pages * page, heads, D)
    j = torch.arange(shape[0], device=device, dtype=torch.float32)[:, None, None]
    d = torch.arange(D, device=device, dtype=torch.float32)
    v = torch.cos(2 * math.pi * j * (d % 7 + 1) / n + d) + 0.3 * torch.randn(shape, generator=gen, device=device)
    k = torch.randn(shape, generator=gen, device=device)
    if not kv:
        return k.to(dtype).view(pages, page, heads, D), v.to(dtype).view(pages, page, heads, D), None, None
    scales = [(torch.rand((pages, heads, page), generator=gen, device=device) * 0.25 + 0.875) * 0.01 for _ in range(2)]
    k, v = ((x.view(pages, page, heads, D) / s.transpose(1, 2)[..., None]).clamp(-448, 448).to(E4M3)
            for x, s in zip((k, v), scales))
    return k, v, *scales


def long_reference(q, n, k, v, ks, vs, dtype, lost=None):
    """(out, lse, tolerance) of one request's query [Hq, D]; `lost`: keys whose values are left out of the sum."""
    Hq, D = q.shape
    Hk = k.shape[2]

    def rows(c, s):
        x = c.float().double()
        return (x if s is None else x * s.double().transpose(1, 2)[..., None]).reshape(-1, Hk, D)[:n]
    kk, vv = rows(k, ks), rows(v, vs)
    s = torch.einsum("hgd,nhd->hgn", q.double().view(Hk, Hq // Hk, D), kk) / math.sqrt(D)
    p = torch.softmax(s, -1)
    w = p.clone()
    if lost is not None:
        w[..., lost] = 0.0
    out = torch.einsum("hgn,nhd->hgd", w, vv)
    weight = UNIT[torch.float16 if ks is not None else dtype]
    tol = 8 * weight * torch.einsum("hgn,nhd->hgd", p * p, vv * vv).sqrt() + UNIT[dtype] * out.abs() \
        + 2.0 ** -16 * torch.einsum("hgn,nhd->hgd", p, vv.abs()) \
        + 2.0 ** -31 * p.amax(-1)[..., None] * vv.abs().sum(0)[:, None] + 2.0 ** -25
    return out.reshape(Hq, D), torch.logsumexp(s, -1).reshape(Hq), tol.reshape(Hq, D)
