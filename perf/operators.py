"""Measured cases of the serving operators: token log probabilities, the paged
key-value append (norm, rotation, quantised write) and paged decode attention.

``run`` computes a case through plain elementary torch operations in float32
(``own = False``) or through the library's entry points (``own = True``);
``exact`` restates each operator in float64 from its definition.
"""
from __future__ import annotations

import functools
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
E4M3_MAX = 448.0
SCALE_MIN = 1e-12
EPS = 1e-6
ROPE_THETA = 1e6


# ------------------------------------------------------------------- cases
def listed():
    return [
        # one streaming request that asked for its token's log probability and 5 alternatives
        dict(name="logprobs-one-request", op="logprobs", rows=1, vocab=151936, dtype="f16", top_n=5, tokens=1,
             temperature=False, masked=0.0),
        # a full decode batch, 20 alternatives each, scored at the request's temperature
        dict(name="logprobs-decode-batch", op="logprobs", rows=128, vocab=151936, dtype="f16", top_n=20, tokens=1,
             temperature=True, masked=0.0),
        # the prompt's own log probabilities: every position of a chunk of prefill
        dict(name="logprobs-prompt", op="logprobs", rows=2048, vocab=128256, dtype="bf16", top_n=1, tokens=1,
             temperature=False, masked=0.0),
        # choices scored under a grammar mask (most of the vocabulary at -inf), float32 logits, odd vocabulary
        dict(name="logprobs-grammar-f32", op="logprobs", rows=37, vocab=32003, dtype="f32", top_n=8, tokens=4,
             temperature=True, masked=0.9),
        # one new token of one request: nothing but latency
        dict(name="append-one-token", op="append", tokens=1, requests=1, context=511, hq=16, hk=2, dim=128,
             page=16, dtype="f16", e4m3=False, norm=False, interleaved=False),
        # a decode batch into an e4m3 cache, heads normalised
        dict(name="append-decode-e4m3", op="append", tokens=128, requests=128, context=384, hq=32, hk=8, dim=128,
             page=16, dtype="bf16", e4m3=True, norm=True, interleaved=False),
        # a large prefill chunk, heads normalised
        dict(name="append-prefill", op="append", tokens=8192, requests=4, context=100, hq=32, hk=8, dim=128,
             page=16, dtype="bf16", e4m3=False, norm=True, interleaved=False),
        # a mixed chunk of odd length, interleaved pairs, small heads, e4m3 cache
        dict(name="append-odd-chunk", op="append", tokens=1001, requests=7, context=333, hq=14, hk=2, dim=64,
             page=32, dtype="f16", e4m3=True, norm=False, interleaved=True),
        # one request at the end of a 128 + 384 token generation
        dict(name="decode-one-request", op="decode", requests=1, low=512, high=512, hq=16, hk=2, dim=128, page=16,
             dtype="f16", e4m3=False),
        # 128 concurrent requests between their first and last generated token
        dict(name="decode-batch", op="decode", requests=128, low=128, high=512, hq=16, hk=2, dim=128, page=16,
             dtype="f16", e4m3=False),
        # few requests with very long contexts
        dict(name="decode-long", op="decode", requests=4, low=100001, high=131072, hq=32, hk=8, dim=128, page=16,
             dtype="bf16", e4m3=False),
        # very uneven lengths over an e4m3 cache
        dict(name="decode-ragged-e4m3", op="decode", requests=64, low=1, high=16384, hq=32, hk=8, dim=128, page=16,
             dtype="bf16", e4m3=True),
    ]


def _log_int(rng, low, high):
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    n = max(low, min(high, n))
    return n + 1 if n == 3072 else n


def draw(rng):
    op = rng.choice(("logprobs", "append", "decode"))
    heads, dim = rng.choice(((16, 2), (32, 8), (14, 2), (28, 4), (8, 8), (40, 2), (5, 1))), rng.choice((64, 128, 128, 256))
    if (heads[0] + 2 * heads[1]) * dim == 3072:
        dim = 128
    if op == "logprobs":
        vocab = rng.choice((151936, 128256, 32003, _log_int(rng, 500, 151936)))
        rows = _log_int(rng, 1, min(2048, 2048 * 128256 // vocab))
        dtype = rng.choice(("f16", "bf16", "f32"))
        if dtype == "f32":
            rows = max(1, rows // 2)
        return dict(op=op, rows=rows, vocab=vocab, dtype=dtype, top_n=rng.choice((0, 1, 5, 8, 20)),
                    tokens=rng.choice((1, 1, 3)), temperature=rng.random() < 0.5,
                    masked=rng.choice((0.0, 0.0, 0.5, 0.99)))
    if op == "append":
        tokens = _log_int(rng, 1, 8192)
        return dict(op=op, tokens=tokens, requests=min(tokens, _log_int(rng, 1, 128)), context=_log_int(rng, 1, 400),
                    hq=heads[0], hk=heads[1], dim=dim if tokens < 4096 else min(dim, 128), page=rng.choice((16, 16, 32, 1, 64)),
                    dtype=rng.choice(("f16", "bf16")), e4m3=rng.random() < 0.5, norm=rng.random() < 0.5,
                    interleaved=rng.random() < 0.3)
    requests = _log_int(rng, 1, 128)
    room = 4 * 131072 * 8 * 128 // (requests * heads[1] * dim)
    high = _log_int(rng, 1, max(1, min(131072, room)))
    return dict(op=op, requests=requests, low=_log_int(rng, 1, high), high=high, hq=heads[0], hk=heads[1], dim=dim,
                page=rng.choice((16, 16, 32, 1, 64)), dtype=rng.choice(("f16", "bf16")), e4m3=rng.random() < 0.5)


def _lengths(case):
    """Lengths of a case's requests, spread over [low, high] by their logarithm; the same for every seed."""
    n, low, high = case["requests"], case["low"], case["high"]
    at = [((i + 1) * 0.6180339887498949) % 1.0 for i in range(n)]
    got = [int(round(math.exp(math.log(low) + a * (math.log(high) - math.log(low))))) for a in at]
    got[0] = high
    return [g + 1 if g == 3072 else g for g in got]


def _chunks(case):
    """New tokens of each request of an append case."""
    n, r = case["tokens"], case["requests"]
    return [n // r + (1 if i < n % r else 0) for i in range(r)]


# ------------------------------------------------------------------ inputs
def _rand(shape, dtype, gen, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _pages(lengths, page, gen):
    """Page lists in the order a pool hands them out: scattered."""
    counts = [-(-n // page) for n in lengths]
    total = sum(counts)
    spare = total // 8 + 1
    order = torch.randperm(total + spare, generator=gen, device="cuda")[:total].to(torch.int32)
    indptr = torch.tensor([0] + counts, dtype=torch.int32).cumsum(0).to(torch.int32).cuda()
    return total + spare, indptr, order


def _empty_cache(pages, case):
    shape = (pages, case["page"], case["hk"], case["dim"])
    kv = torch.float8_e4m3fn if case["e4m3"] else DTYPES[case["dtype"]]
    size = 1 if case["e4m3"] else 2
    k, v = (torch.zeros(math.prod(shape) * size, dtype=torch.uint8, device="cuda").view(kv).view(shape) for _ in range(2))
    if not case["e4m3"]:
        return k, v, None, None
    s = (pages, case["hk"], case["page"])
    return k, v, torch.zeros(s, device="cuda"), torch.zeros(s, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    if case["op"] == "logprobs":
        R, V, dt = case["rows"], case["vocab"], DTYPES[case["dtype"]]
        # a row of a language model's logits: a broad bulk and a few likely tokens
        x = _rand((R, V), dt, gen, 2.5)
        spikes = torch.randint(0, V, (R, 1), generator=gen, device="cuda")
        spikes = (spikes + torch.arange(8, device="cuda") * (V // 8)) % V
        x.scatter_(1, spikes, _rand((R, 8), dt, gen, 2.0) + 9.0)
        if case["masked"]:
            gone = torch.rand((R, V), generator=gen, device="cuda") < case["masked"]
            gone.scatter_(1, spikes[:, :4], False)
            x.masked_fill_(gone, float("-inf"))
        tok = torch.randint(0, V, (R, case["tokens"]), generator=gen, device="cuda", dtype=torch.int32)
        tok[:, 0] = spikes[:, 0].to(torch.int32)
        s.update(logits=x, token_ids=tok, temps=None)
        if case["temperature"]:
            s["temps"] = torch.rand(R, generator=gen, device="cuda") * 0.7 + 0.5
        return s
    hq, hk, D, dt = case["hq"], case["hk"], case["dim"], DTYPES[case["dtype"]]
    if case["op"] == "append":
        new = _chunks(case)
        lengths = [case["context"] + c for c in new]
        pages, indptr, indices = _pages(lengths, case["page"], gen)
        T = case["tokens"]
        qkv = _rand((T, (hq + 2 * hk) * D), dt, gen, 1.5)
        b = torch.repeat_interleave(torch.arange(len(new), dtype=torch.int32), torch.tensor(new))
        first = torch.tensor([0] + new).cumsum(0)[:-1]
        pos = (torch.arange(T) - first[b.long()] + case["context"]).to(torch.int32)
        if T > 8:
            b[-1] = -1  # a padding row of a captured batch
        inv = ROPE_THETA ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
        ang = (torch.arange(max(lengths), dtype=torch.float64)[:, None] * inv[None, :]).cuda()
        s["cos_sin"] = torch.cat([ang.cos(), ang.sin()], 1).float()
        s["qkv"] = qkv
        s["batch_index"], s["positions"] = b.cuda(), pos.cuda()
        s["q_norm"] = s["k_norm"] = None
        if case["norm"]:
            s["q_norm"], s["k_norm"] = _rand((D,), dt, gen, 0.2) + 1, _rand((D,), dt, gen, 0.2) + 1
        s["q_out"] = torch.empty((T, hq, D), dtype=dt, device="cuda")
        s["k"], s["v"], s["ks"], s["vs"] = _empty_cache(pages, case)
    else:
        lengths = _lengths(case)
        order = torch.randperm(len(lengths), generator=gen, device="cuda").tolist()
        lengths = [lengths[i] for i in order]
        pages, indptr, indices = _pages(lengths, case["page"], gen)
        s["k"], s["v"], s["ks"], s["vs"] = _empty_cache(pages, case)
        for name, scale in (("k", "ks"), ("v", "vs")):
            c = s[name]
            step = max(1, (1 << 26) // max(1, c[0].numel()))
            for at in range(0, pages, step):
                part = _rand(c[at:at + step].shape, torch.float32, gen)
                if case["e4m3"]:  # as the append leaves it: the largest magnitude of each token and head at 448
                    sc = part.abs().amax(-1).clamp_min(SCALE_MIN) / E4M3_MAX
                    s[scale][at:at + step] = sc.transpose(1, 2)
                    part = part / sc[..., None]
                c[at:at + step] = part.to(c.dtype)
        # scores of a standard deviation of 2: attention that prefers some keys
        s["q"] = _rand((len(lengths), hq, D), dt, gen, 2.0)
        s["last"] = torch.tensor([(n - 1) % case["page"] + 1 for n in lengths], dtype=torch.int32).cuda()
        s["max_len"] = max(lengths)
    s["indptr"], s["indices"] = indptr, indices
    return s


# -------------------------------------------------------------- plain forms
def _plain_logprobs(s):
    x = s["logits"].float()
    R, V = x.shape
    temp = torch.ones(R, device=x.device) if s["temps"] is None else s["temps"]
    m = x.amax(1, keepdim=True)
    z = (x - m) / temp[:, None]
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    lz = torch.log(total)
    entropy = (lz - torch.where(e > 0, e * z, 0.0).sum(1, keepdim=True) / total)[:, 0]
    picked = z.gather(1, s["token_ids"].long()) - lz
    n = s["top_n"]
    ids = torch.argsort(x, dim=1, descending=True, stable=True)[:, :n]
    top = z.gather(1, ids) - lz
    ids = torch.where(torch.isinf(top), -1, ids)
    return {"logprobs": picked, "entropy": entropy, "top_ids": ids.to(torch.int32), "top_logprobs": top}


def _plain_norm_rotate(x, weight, c, sn, interleaved):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * c - b * sn, b * c + a * sn], -1).flatten(-2)
    a, b = x.chunk(2, -1)
    return torch.cat([a * c - b * sn, b * c + a * sn], -1)


def _plain_append(s):
    hq, hk, D, page = s["hq"], s["hk"], s["dim"], s["page"]
    q, k, v = (t.reshape(t.shape[0], -1, D) for t in s["qkv"].split([hq * D, hk * D, hk * D], 1))
    c, sn = s["cos_sin"][s["positions"].long()][:, None, :].chunk(2, -1)
    s["q_out"].copy_(_plain_norm_rotate(q, s["q_norm"], c, sn, s["interleaved"]))
    k = _plain_norm_rotate(k, s["k_norm"], c, sn, s["interleaved"])
    keep = s["batch_index"] >= 0
    b, pos = s["batch_index"][keep].long(), s["positions"][keep].long()
    at = s["indices"][s["indptr"][b].long() + pos // page].long()
    k, v, slot = k[keep], v[keep].float(), pos % page
    if s["ks"] is not None:
        sk, sv = (t.abs().amax(-1).clamp_min(SCALE_MIN * E4M3_MAX) / E4M3_MAX for t in (k, v))
        s["ks"][at, :, slot], s["vs"][at, :, slot] = sk, sv
        k, v = k / sk[..., None], v / sv[..., None]
        # rounded to e4m3 by the type's own conversion; the cache is indexed through its bytes
        s["k"].view(torch.uint8)[at, slot] = k.to(torch.float8_e4m3fn).view(torch.uint8)
        s["v"].view(torch.uint8)[at, slot] = v.to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        s["k"][at, slot], s["v"][at, slot] = k.to(s["k"].dtype), v.to(s["v"].dtype)
    return _append_outputs(s)


def _append_outputs(s):
    out = {"q": s["q_out"], "k_cache": s["k"], "v_cache": s["v"]}
    if s["ks"] is not None:
        out.update(k_scale=s["ks"], v_scale=s["vs"])
    return out


def _plain_decode(s):
    hq, hk, D, page = s["hq"], s["hk"], s["dim"], s["page"]
    indptr = s["indptr"].long()
    B = indptr.numel() - 1
    length = (indptr[1:] - indptr[:-1] - 1) * page + s["last"]
    j = torch.arange(s["max_len"], device="cuda")
    live = j[None, :] < length[:, None]
    at = (indptr[:-1, None] + j[None, :] // page).clamp_max(s["indices"].numel() - 1)
    at, slot = s["indices"][at].long(), (j % page)[None, :].expand(B, -1)

    def read(c, scale):
        # [B, len, Hk, D] in float32, through the bytes where the type has no indexing of its own
        x = c.view(torch.uint8)[at, slot].view(torch.float8_e4m3fn).float() if scale is not None else c[at, slot].float()
        return x if scale is None else x * scale[at, :, slot][..., None]

    q = s["q"].float().reshape(B, hk, hq // hk, D)
    score = (read(s["k"], s["ks"]).permute(0, 2, 1, 3) @ q.transpose(-1, -2)).transpose(-1, -2) / math.sqrt(D)
    score.masked_fill_(~live[:, None, None, :], float("-inf"))
    m = score.amax(-1, keepdim=True)
    p = torch.exp(score - m)
    total = p.sum(-1, keepdim=True)
    out = (p / total) @ read(s["v"], s["vs"]).permute(0, 2, 1, 3)
    lse = (m + torch.log(total))[..., 0]
    return {"out": out.reshape(B, hq, D).to(s["q"].dtype), "lse": lse.reshape(B, hq)}


# ------------------------------------------------------------------ own form
# What a serving program makes once and keeps for all its steps: the handles with their workspaces.
@functools.lru_cache(maxsize=None)
def _scorer(vocab, dtype):
    from ecahlang_b200.logprobs import TokenLogprobs
    return TokenLogprobs(vocab, DTYPES[dtype])


@functools.lru_cache(maxsize=None)
def _attention(hq, hk, dim, page, dtype, e4m3):
    from ecahlang_b200.paged import PagedAttention
    return PagedAttention(hq, hk, dim, page, DTYPES[dtype], kv_dtype=torch.float8_e4m3fn if e4m3 else None,
                          max_batch=128)


def _own(s):
    if s["op"] == "logprobs":
        r = _scorer(s["vocab"], s["dtype"])(s["logits"], s["token_ids"], top_n=s["top_n"], temperature=s["temps"])
        return {"logprobs": r.logprobs, "entropy": r.entropy, "top_ids": r.top_ids, "top_logprobs": r.top_logprobs}
    att = _attention(s["hq"], s["hk"], s["dim"], s["page"], s["dtype"], s["e4m3"])
    if s["op"] == "append":
        hq, hk, D = s["hq"], s["hk"], s["dim"]
        q, k, v = s["qkv"].view(-1, hq + 2 * hk, D).split([hq, hk, hk], 1)
        att.append(q, k, v, s["positions"], s["batch_index"], s["indptr"], s["indices"], s["k"], s["v"],
                   k_scale=s["ks"], v_scale=s["vs"], cos_sin=s["cos_sin"], q_norm=s["q_norm"], k_norm=s["k_norm"],
                   eps=EPS, interleaved=s["interleaved"], q_out=s["q_out"])
        return _append_outputs(s)
    out, lse = att.decode(s["q"], s["indptr"], s["indices"], s["last"], s["k"], s["v"], k_scale=s["ks"],
                          v_scale=s["vs"], return_lse=True)
    return {"out": out, "lse": lse}


def run(state):
    if own:
        return _own(state)
    return {"logprobs": _plain_logprobs, "append": _plain_append, "decode": _plain_decode}[state["op"]](state)


# ------------------------------------------------------------------- work
def work(case):
    if case["op"] == "logprobs":
        R, V = case["rows"], case["vocab"]
        size = 4 if case["dtype"] == "f32" else 2
        return {"bytes": R * V * size + R * (4 + 8 * case["tokens"] + 8 * case["top_n"] + (4 if case["temperature"] else 0)),
                "flops": 6 * R * V}
    hq, hk, D, kv = case["hq"], case["hk"], case["dim"], 1 if case["e4m3"] else 2
    scales = 8 * hk if case["e4m3"] else 0
    if case["op"] == "append":
        T = case["tokens"]
        table = 4 * D * min(T, max(_chunks(case)))
        return {"bytes": T * ((2 * hq + 2 * hk) * D * 2 + 2 * hk * D * kv + scales + 8) + table, "flops": 10 * T * (hq + 2 * hk) * D}
    n = sum(_lengths(case))
    B = case["requests"]
    return {"bytes": n * (2 * hk * D * kv + scales) + B * hq * (4 * D + 4) + 4 * -(-n // case["page"]), "flops": 4 * n * hq * D}


# ------------------------------------------------------------------- exact
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logprobs":
        got = {"logprobs": [], "entropy": [], "top_logprobs": []}
        for at in range(0, case["rows"], 256):
            x = s["logits"][at:at + 256].double()
            if s["temps"] is not None:
                x = x / s["temps"][at:at + 256].double()[:, None]
            lp = x - torch.logsumexp(x, 1, keepdim=True)
            got["logprobs"].append(torch.gather(lp, 1, s["token_ids"][at:at + 256].long()))
            got["entropy"].append(torch.special.entr(lp.exp()).sum(1))
            got["top_logprobs"].append(torch.topk(lp, case["top_n"], dim=1).values)
        return {"logprobs": torch.cat(got["logprobs"]), "entropy": torch.cat(got["entropy"]), "top_ids": None,
                "top_logprobs": torch.cat(got["top_logprobs"])}
    if case["op"] == "append":
        hq, hk, D, page = case["hq"], case["hk"], case["dim"], case["page"]
        x = s["qkv"].double().view(-1, hq + 2 * hk, D)
        table = torch.complex(s["cos_sin"][:, :D // 2].double(), s["cos_sin"][:, D // 2:].double())

        def turn(h, w):
            if w is not None:
                h = h / torch.sqrt(h.pow(2).mean(-1, keepdim=True) + EPS) * w.double()
            r = table[s["positions"].long()][:, None, :]
            if case["interleaved"]:
                return torch.view_as_real(torch.view_as_complex(h.reshape(*h.shape[:-1], D // 2, 2).contiguous()) * r).flatten(-2)
            z = torch.complex(h[..., :D // 2].contiguous(), h[..., D // 2:].contiguous()) * r
            return torch.cat([z.real, z.imag], -1)

        out = {"q": turn(x[:, :hq], s["q_norm"])}
        flat = {}
        rows = [i for i, b in enumerate(s["batch_index"].tolist()) if b >= 0]
        b, pos = s["batch_index"].tolist(), s["positions"].tolist()
        indptr, indices = s["indptr"].tolist(), s["indices"].tolist()
        at = torch.tensor([indices[indptr[b[i]] + pos[i] // page] * page + pos[i] % page for i in rows], device="cuda")
        for name, h in (("k", turn(x[:, hq:hq + hk], s["k_norm"])), ("v", x[:, hq + hk:])):
            c = s[name]
            h = h[rows]
            if case["e4m3"]:
                sc = h.abs().amax(-1).clamp_min(SCALE_MIN * E4M3_MAX) / E4M3_MAX
                scales = torch.zeros((c.shape[0] * page, hk), dtype=torch.float64, device="cuda")
                scales[at] = sc
                flat[name + "_scale"] = scales.view(c.shape[0], page, hk).transpose(1, 2).contiguous()
                h = h / sc[..., None]
            cache = torch.zeros((c.shape[0] * page, hk, D), dtype=torch.float64, device="cuda")
            cache[at] = h
            flat[name + "_cache"] = cache.view(c.shape)
        return out | flat
    hq, hk, D, page = case["hq"], case["hk"], case["dim"], case["page"]
    outs, lses = [], []
    indptr, last = s["indptr"].tolist(), s["last"].tolist()
    for b in range(case["requests"]):
        pages = s["indices"][indptr[b]:indptr[b + 1]].long()
        n = (len(pages) - 1) * page + last[b]
        kv = []
        for c, sc in ((s["k"], s["ks"]), (s["v"], s["vs"])):
            x = c.view(torch.uint8)[pages].view(c.dtype).double() if sc is not None else c[pages].double()
            if sc is not None:
                x = x * sc[pages].double().transpose(1, 2)[..., None]
            kv.append(x.reshape(-1, hk, D)[:n])
        q = s["q"][b].double().view(hk, hq // hk, D)
        logit = torch.einsum("hgd,nhd->hgn", q, kv[0]) / D ** 0.5
        lses.append(torch.logsumexp(logit, -1).reshape(hq))
        outs.append(torch.einsum("hgn,nhd->hgd", torch.softmax(logit, -1), kv[1]).reshape(hq, D))
    return {"out": torch.stack(outs), "lse": torch.stack(lses)}
