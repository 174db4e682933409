"""Measured cases of the operators that serve several new tokens a request: paged
prefill attention, verification of drafted tokens, copies of cache pages.

``run`` computes a case through plain elementary torch operations (``own =
False``) or through the library's entry points (``own = True``); ``exact``
restates each operator in float64 from its definition.
"""
from __future__ import annotations

import functools
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
E4M3_MAX = 448.0
SCALE_MIN = 1e-12


# ------------------------------------------------------------------- cases
def listed():
    return [
        # one short prompt of odd length: nothing but latency
        dict(name="prefill-short-prompt", op="prefill", requests=1, new_low=37, new_high=37, ctx_low=0, ctx_high=0,
             hq=16, hk=2, dim=128, page=16, dtype="f16", e4m3=False, causal=True),
        # prompts that arrive together, packed without padding
        dict(name="prefill-packed-prompts", op="prefill", requests=16, new_low=100, new_high=1024, ctx_low=0, ctx_high=0,
             hq=16, hk=2, dim=128, page=16, dtype="f16", e4m3=False, causal=True),
        # one long prompt
        dict(name="prefill-long-prompt", op="prefill", requests=1, new_low=8192, new_high=8192, ctx_low=0, ctx_high=0,
             hq=32, hk=8, dim=128, page=16, dtype="bf16", e4m3=False, causal=True),
        # chunks of prompts behind contexts that an e4m3 cache holds
        dict(name="prefill-chunks-e4m3", op="prefill", requests=7, new_low=90, new_high=333, ctx_low=1000, ctx_high=6001,
             hq=32, hk=8, dim=128, page=16, dtype="bf16", e4m3=True, causal=True),
        # a draft of four and the token before it, for a batch of very uneven contexts
        dict(name="prefill-drafts", op="prefill", requests=64, new_low=5, new_high=5, ctx_low=10, ctx_high=8000,
             hq=32, hk=8, dim=128, page=16, dtype="bf16", e4m3=False, causal=True),
        # wide heads without groups, pages of one token, every key visible
        dict(name="prefill-wide-heads", op="prefill", requests=2, new_low=701, new_high=1500, ctx_low=0, ctx_high=64,
             hq=8, hk=8, dim=256, page=1, dtype="f16", e4m3=False, causal=False),
        # one streaming request with a draft of four
        dict(name="verify-one-request", op="verify", requests=1, drafts=4, vocab=151936, dtype="f32", given=True,
             ragged=False, kept=1.0, near=0.5),
        # a batch whose draft and target distributions are what top-k and top-p left
        dict(name="verify-batch", op="verify", requests=64, drafts=5, vocab=151936, dtype="f32", given=True,
             ragged=False, kept=0.01, near=0.5),
        # drafts looked up in the prompt (no distribution of their own), ragged, an odd vocabulary
        dict(name="verify-looked-up", op="verify", requests=128, drafts=8, vocab=32003, dtype="bf16", given=False,
             ragged=True, kept=1.0, near=0.2),
        # a request forks into four choices: its last page, partly filled, copied in all layers
        dict(name="copy-fork", op="copy", pairs=3, pages=64, layers=28, hk=2, dim=128, page=16, dtype="f16",
             e4m3=False, partial=True),
        # a pool compacted: many whole pages move
        dict(name="copy-compact", op="copy", pairs=2000, pages=4096, layers=4, hk=8, dim=128, page=16, dtype="bf16",
             e4m3=False, partial=False),
        # forks of a whole batch over an e4m3 cache with its scales, pages of another size
        dict(name="copy-fork-batch-e4m3", op="copy", pairs=127, pages=512, layers=7, hk=4, dim=64, page=32, dtype="bf16",
             e4m3=True, partial=True),
    ]


def _log_int(rng, low, high):
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return max(low, min(high, n))


def draw(rng):
    op = rng.choice(("prefill", "prefill", "verify", "copy"))
    heads, dim = rng.choice(((16, 2), (32, 8), (14, 2), (28, 4), (8, 8), (40, 2), (5, 1))), rng.choice((64, 96, 128, 128, 192, 256))
    page = rng.choice((16, 16, 32, 1, 64))
    if op == "prefill":
        requests, new = _log_int(rng, 1, 64), _log_int(rng, 1, 8192)
        work, held = 8192 * 8192 * 32 * 128, 64 * 8192 * 8 * 128
        while requests > 1 and (requests * new * new * heads[0] * dim > work or requests * new * heads[1] * dim > held):
            requests //= 2
        if new * new * heads[0] * dim > work:
            heads, dim = (16, 2), 128
        most = min(work // (requests * new * heads[0] * dim), held // (requests * heads[1] * dim), 65536) - new
        context = _log_int(rng, 1, most) if most > 1 and rng.random() < 0.6 else 0
        return dict(op=op, requests=requests, new_low=_log_int(rng, 1, new), new_high=new, ctx_low=context // 3, ctx_high=context,
                    hq=heads[0], hk=heads[1], dim=dim, page=page, dtype=rng.choice(("f16", "bf16")), e4m3=rng.random() < 0.4,
                    causal=rng.random() < 0.8)
    if op == "verify":
        vocab = rng.choice((151936, 128256, 32003, _log_int(rng, 500, 151936)))
        drafts = _log_int(rng, 1, 8)
        requests = _log_int(rng, 1, max(1, min(128, 64 * 6 * 151936 // (vocab * (drafts + 1)))))
        return dict(op=op, requests=requests, drafts=drafts, vocab=vocab, dtype=rng.choice(("f32", "f32", "f16", "bf16")),
                    given=rng.random() < 0.7, ragged=rng.random() < 0.5, kept=rng.choice((1.0, 0.1, 0.01)),
                    near=rng.choice((0.1, 0.5, 1.5)))
    layers = _log_int(rng, 1, 30)
    row = layers * page * heads[1] * dim
    pairs = _log_int(rng, 1, max(1, min(4000, 2000 * 4 * 16 * 8 * 128 // row)))
    return dict(op=op, pairs=pairs, pages=2 * pairs + rng.randrange(1, 100), layers=layers, hk=heads[1], dim=dim, page=page,
                dtype=rng.choice(("f16", "bf16")), e4m3=rng.random() < 0.4, partial=rng.random() < 0.5)


def _spread(n, low, high, phase):
    """n whole numbers spread over [low, high] by their logarithm, the highest among them; the same for every seed."""
    at = [((i + phase) * 0.6180339887498949) % 1.0 for i in range(n)]
    got = [int(round(math.exp(math.log(low + 1) + a * (math.log(high + 1) - math.log(low + 1))))) - 1 for a in at]
    got[0] = high
    return got


def _lengths(case):
    """(new tokens, tokens in all) of each request of a prefill case."""
    new = _spread(case["requests"], case["new_low"], case["new_high"], 1)
    ctx = _spread(case["requests"], case["ctx_low"], case["ctx_high"], 2)
    return new, [a + b for a, b in zip(new, ctx)]


# ------------------------------------------------------------------ inputs
def _rand(shape, dtype, gen, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _fill(cache, scales, gen):
    """Random keys or values; in an e4m3 cache as the append leaves them: the largest magnitude of each token and head at 448."""
    step = max(1, (1 << 26) // max(1, cache[0].numel()))
    for at in range(0, cache.shape[0], step):
        part = _rand(cache[at:at + step].shape, torch.float32, gen)
        if scales is not None:
            sc = part.abs().amax(-1).clamp_min(SCALE_MIN) / E4M3_MAX
            scales[at:at + step] = sc.transpose(1, 2)
            part = part / sc[..., None]
        cache[at:at + step] = part.to(cache.dtype)


def _cache(pages, case, gen):
    """(k, v, k_scale, v_scale): [pages, page, heads, dim] and, for e4m3, scales [pages, heads, page]."""
    shape = (pages, case["page"], case["hk"], case["dim"])
    kv = torch.float8_e4m3fn if case["e4m3"] else DTYPES[case["dtype"]]
    k, v = (torch.zeros(math.prod(shape) * kv.itemsize, dtype=torch.uint8, device="cuda").view(kv).view(shape) for _ in range(2))
    ks = vs = None
    if case["e4m3"]:
        ks, vs = (torch.zeros((pages, case["hk"], case["page"]), device="cuda") for _ in range(2))
    _fill(k, ks, gen)
    _fill(v, vs, gen)
    return k, v, ks, vs


def _prepare_prefill(s, gen):
    new, lengths = _lengths(s)
    order = torch.randperm(len(new), generator=gen, device="cuda").tolist()
    new, lengths = [new[i] for i in order], [lengths[i] for i in order]
    page = s["page"]
    counts = [-(-n // page) for n in lengths]
    total = sum(counts)
    s["k"], s["v"], s["ks"], s["vs"] = _cache(total + total // 8 + 1, s, gen)
    # page lists in the order a pool hands them out: scattered
    s["indices"] = torch.randperm(s["k"].shape[0], generator=gen, device="cuda")[:total].to(torch.int32)
    s["indptr"] = torch.tensor([0] + counts).cumsum(0).to(torch.int32).cuda()
    s["last"] = torch.tensor([(n - 1) % page + 1 for n in lengths], dtype=torch.int32).cuda()
    s["qo_indptr"] = torch.tensor([0] + new).cumsum(0).to(torch.int32).cuda()
    # scores of a standard deviation of 2: attention that prefers some keys
    s["q"] = _rand((sum(new), s["hq"], s["dim"]), DTYPES[s["dtype"]], gen, 2.0)
    s["max_new"], s["max_len"] = max(new), max(lengths)


def _prepare_verify(s, gen):
    B, N, V, dt = s["requests"], s["drafts"], s["vocab"], DTYPES[s["dtype"]]
    # a language model's logits: a broad bulk and a few likely tokens; the draft model's are near the target's
    x = torch.randn((B, N + 1, V), generator=gen, device="cuda") * 2.5
    spikes = torch.randint(0, V, (B, N + 1, 8), generator=gen, device="cuda")
    x.scatter_(2, spikes, torch.randn((B, N + 1, 8), generator=gen, device="cuda") * 2.0 + 11.0)
    y = x[:, :N] + torch.randn((B, N, V), generator=gen, device="cuda") * s["near"]

    def probabilities(z):
        if s["kept"] < 1.0:  # what top-k leaves
            least = torch.topk(z, max(1, int(V * s["kept"])), dim=-1).values[..., -1:]
            z = z.masked_fill(z < least, float("-inf"))
        return torch.softmax(z, -1)

    s["target"] = probabilities(x).to(dt)
    y = probabilities(y)
    s["draft_ids"] = torch.multinomial(y.view(B * N, V), 1, generator=gen).view(B, N).to(torch.int32)
    s["draft"] = y.to(dt) if s["given"] else None
    s["uniforms"] = torch.rand((B, N + 1), generator=gen, device="cuda")
    s["num_drafts"] = torch.randint(0, N + 1, (B,), generator=gen, device="cuda", dtype=torch.int32) if s["ragged"] else None


def _prepare_copy(s, gen):
    L, pages, page = s["layers"], s["pages"], s["page"]
    kv = torch.float8_e4m3fn if s["e4m3"] else DTYPES[s["dtype"]]
    shape = (L, pages, page, s["hk"], s["dim"])
    s["ks"] = s["vs"] = None
    s["k"], s["v"] = (torch.zeros(math.prod(shape) * kv.itemsize, dtype=torch.uint8, device="cuda").view(kv).view(shape) for _ in range(2))
    if s["e4m3"]:
        s["ks"], s["vs"] = (torch.zeros((L, pages, s["hk"], page), device="cuda") for _ in range(2))
    for i in range(L):
        for c, sc in ((s["k"], s["ks"]), (s["v"], s["vs"])):
            _fill(c[i], None if sc is None else sc[i], gen)
    # what the program keeps: one cache a layer
    s["caches"] = [(s["k"][i], s["v"][i], s["ks"][i] if s["e4m3"] else None, s["vs"][i] if s["e4m3"] else None) for i in range(L)]
    at = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    n = s["pairs"]
    s["dst"] = at[:n].contiguous()
    s["src"] = at[n:2 * n].contiguous()
    s["tokens"] = None
    if s["partial"]:
        s["src"] = s["src"][torch.arange(n, device="cuda") // 3 * 3]  # a page goes to up to three children
        s["tokens"] = torch.randint(1, page + 1, (n,), generator=gen, device="cuda", dtype=torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    {"prefill": _prepare_prefill, "verify": _prepare_verify, "copy": _prepare_copy}[case["op"]](s, gen)
    return s


# -------------------------------------------------------------- plain forms
def _plain_prefill(s):
    hq, hk, D, page = s["hq"], s["hk"], s["dim"], s["page"]
    indptr, qptr = s["indptr"].long(), s["qo_indptr"].long()
    B, T = indptr.numel() - 1, s["q"].shape[0]
    length = (indptr[1:] - indptr[:-1] - 1) * page + s["last"]
    new = qptr[1:] - qptr[:-1]
    j = torch.arange(s["max_len"], device="cuda")
    at = (indptr[:-1, None] + j[None, :] // page).clamp_max(s["indices"].numel() - 1)
    at, slot = s["indices"][at].long(), (j % page)[None, :].expand(B, -1)

    def read(c, scale):
        # [B, Hk, len, D] in float32, through the bytes where the type has no indexing of its own
        x = c.view(torch.uint8)[at, slot].view(torch.float8_e4m3fn).float() if scale is not None else c[at, slot].float()
        return (x if scale is None else x * scale[at, :, slot][..., None]).permute(0, 2, 1, 3)

    # queries padded to the longest request: [B, Hk, G, n, D]
    i = torch.arange(s["max_new"], device="cuda")
    row = (qptr[:-1, None] + i[None, :]).clamp_max(T - 1)
    q = s["q"][row].float().view(B, -1, hk, hq // hk, D).permute(0, 2, 3, 1, 4)
    score = (q.reshape(B, hk, -1, D) @ read(s["k"], s["ks"]).transpose(-1, -2)).view(B, hk, hq // hk, -1, s["max_len"])
    score *= 1.0 / math.sqrt(D)
    seen = (length - new)[:, None] + i[None, :] if s["causal"] else (length - 1)[:, None].expand(-1, s["max_new"])
    score.masked_fill_((j[None, None, :] > seen[:, :, None])[:, None, None], float("-inf"))
    m = score.amax(-1, keepdim=True)
    m = torch.where(torch.isinf(m), 0.0, m)
    p = score.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    lse = (m + torch.log(total))[..., 0]
    p /= torch.where(total == 0, 1.0, total)
    out = p.view(B, hk, -1, s["max_len"]) @ read(s["v"], s["vs"])
    out = out.view(B, hq, -1, D).transpose(1, 2)
    b = torch.repeat_interleave(torch.arange(B, device="cuda"), new, output_size=T)
    n = torch.arange(T, device="cuda") - qptr[b]
    return {"out": out[b, n].to(s["q"].dtype), "lse": lse.view(B, hq, -1)[b, :, n].contiguous()}


def _plain_verify(s):
    B, N, V = s["requests"], s["drafts"], s["vocab"]
    x, u = s["draft_ids"].long(), s["uniforms"].double()
    n = torch.full((B,), N, device="cuda") if s["num_drafts"] is None else s["num_drafts"].long()
    px = s["target"][:, :N].gather(2, x[..., None])[..., 0].double()
    qx = torch.ones_like(px) if s["draft"] is None else s["draft"].gather(2, x[..., None])[..., 0].double()
    j = torch.arange(N, device="cuda")
    ok = (u[:, :N] * qx < px) & (j[None, :] < n[:, None])
    accepted = ok.long().cumprod(1).sum(1)
    refused = accepted < n
    b = torch.arange(B, device="cuda")
    p = s["target"][b, accepted].float()
    at = accepted.clamp_max(N - 1)
    if s["draft"] is None:
        q = torch.zeros_like(p).scatter_(1, x[b, at][:, None], float("inf"))
    else:
        q = s["draft"][b, at].float()
    r = torch.where(refused[:, None], (p - q).clamp_min(0.0), p)
    r = torch.where(r.sum(1, keepdim=True) > 0, r, p)
    c = r.double().cumsum(1)
    token = (c <= u[:, N:] * c[:, -1:]).sum(1)
    token = torch.where(c[:, -1] > 0, token, -1)
    k = torch.arange(N + 1, device="cuda")[None, :]
    drafts = torch.cat([x, x.new_full((B, 1), -1)], 1)
    tokens = torch.where(k < accepted[:, None], drafts, torch.where(k == accepted[:, None], token[:, None], -1))
    return {"tokens": tokens.to(torch.int32), "accepted": accepted.to(torch.int32)}


def _plain_copy(s):
    src, dst = s["src"].long(), s["dst"].long()
    slots = torch.arange(s["page"], device="cuda")
    live = None if s["tokens"] is None else (slots[None, :] < s["tokens"][:, None])

    def move(c, mask):
        c = c.view(torch.uint8) if c.dtype.itemsize == 1 else c
        c[:, dst] = c[:, src] if mask is None else torch.where(mask, c[:, src], c[:, dst])

    move(s["k"], None if live is None else live[None, :, :, None, None])
    move(s["v"], None if live is None else live[None, :, :, None, None])
    if s["ks"] is not None:
        move(s["ks"], None if live is None else live[None, :, None, :])
        move(s["vs"], None if live is None else live[None, :, None, :])
    return _copied(s)


def _copied(s):
    out = {"k": s["k"], "v": s["v"]}
    if s["ks"] is not None:
        out.update(k_scale=s["ks"], v_scale=s["vs"])
    return out


# ------------------------------------------------------------------ own form
# What a serving program makes once and keeps for all its steps: the handles with their workspaces.
@functools.lru_cache(maxsize=None)
def _attention(hq, hk, dim, page, dtype, e4m3):
    from ecahlang_b200.paged import PagedAttention
    return PagedAttention(hq, hk, dim, page, DTYPES[dtype], kv_dtype=torch.float8_e4m3fn if e4m3 else None,
                          max_batch=128)


@functools.lru_cache(maxsize=None)
def _verifier(vocab):
    from ecahlang_b200.drafts import DraftVerifier
    return DraftVerifier(vocab, max_batch=128)


def _own(s):
    if s["op"] == "verify":
        r = _verifier(s["vocab"])(s["target"], s["draft_ids"], s["uniforms"], draft_probs=s["draft"], num_drafts=s["num_drafts"])
        return {"tokens": r.tokens, "accepted": r.accepted}
    if s["op"] == "copy":
        att = _attention(s["hk"], s["hk"], s["dim"], s["page"], s["dtype"], s["e4m3"])
        att.copy_pages(s["src"], s["dst"], s["caches"], tokens=s["tokens"])
        return _copied(s)
    att = _attention(s["hq"], s["hk"], s["dim"], s["page"], s["dtype"], s["e4m3"])
    out, lse = att.prefill(s["q"], s["qo_indptr"], s["indptr"], s["indices"], s["last"], s["k"], s["v"], k_scale=s["ks"],
                           v_scale=s["vs"], causal=s["causal"], return_lse=True)
    return {"out": out, "lse": lse}


def run(state):
    if own:
        return _own(state)
    return {"prefill": _plain_prefill, "verify": _plain_verify, "copy": _plain_copy}[state["op"]](state)


# ------------------------------------------------------------------- work
def work(case):
    if case["op"] == "verify":
        B, N, V = case["requests"], case["drafts"], case["vocab"]
        size = 4 if case["dtype"] == "f32" else 2
        # the target's row where a request stops, and the draft's where it has one and was refused (nearly always)
        rows = B * (2 if case["given"] else 1)
        return {"bytes": rows * V * size + B * (N * (4 + 2 * size) + 8 * (N + 1) + 8), "flops": 3 * rows * V}
    if case["op"] == "copy":
        token = case["hk"] * (case["dim"] * 2 * (1 if case["e4m3"] else 2) + (8 if case["e4m3"] else 0))
        n = case["pairs"] * case["layers"] * case["page"] * (0.5 + 0.5 / case["page"] if case["partial"] else 1.0)
        return {"bytes": 2 * n * token + 12 * case["pairs"], "flops": 0}
    hq, hk, D = case["hq"], case["hk"], case["dim"]
    new, lengths = _lengths(case)
    held = sum(lengths) * hk * (2 * D * (1 if case["e4m3"] else 2) + (8 if case["e4m3"] else 0))
    seen = sum(n * (n + 1) // 2 + n * (c - n) if case["causal"] else n * c for n, c in zip(new, lengths))
    return {"bytes": held + sum(new) * hq * (4 * D + 4) + 4 * sum(-(-n // case["page"]) for n in lengths),
            "flops": 4 * D * hq * seen}


# ------------------------------------------------------------------- exact
def exact(case, seed):
    if case["op"] == "verify":
        return None  # whole numbers alone
    s = prepare(case, seed)
    if case["op"] == "copy":
        got = {}
        src, dst = s["src"].tolist(), s["dst"].tolist()
        tokens = s["tokens"].tolist() if s["partial"] else [case["page"]] * len(src)
        for name, c in (("k", s["k"]), ("v", s["v"]), ("k_scale", s["ks"]), ("v_scale", s["vs"])):
            if c is None:
                continue
            x = c.double()
            for a, b, n in zip(src, dst, tokens):
                if name.endswith("scale"):
                    x[:, b, :, :n] = x[:, a, :, :n]
                else:
                    x[:, b, :n] = x[:, a, :n]
            got[name] = x
        return got
    hq, hk, D, page = case["hq"], case["hk"], case["dim"], case["page"]
    T = s["q"].shape[0]
    out = torch.zeros((T, hq, D), dtype=torch.float64, device="cuda")
    lse = torch.full((T, hq), -math.inf, dtype=torch.float64, device="cuda")
    indptr, qptr, last = s["indptr"].tolist(), s["qo_indptr"].tolist(), s["last"].tolist()
    for b in range(case["requests"]):
        pages = s["indices"][indptr[b]:indptr[b + 1]].long()
        n, m = (len(pages) - 1) * page + last[b], qptr[b + 1] - qptr[b]
        kv = []
        for c, sc in ((s["k"], s["ks"]), (s["v"], s["vs"])):
            x = c.view(torch.uint8)[pages].view(c.dtype).double() if sc is not None else c[pages].double()
            if sc is not None:
                x = x * sc[pages].double().transpose(1, 2)[..., None]
            kv.append(x.reshape(-1, hk, D)[:n])
        for at in range(0, m, 512):
            rows = slice(qptr[b] + at, min(qptr[b] + at + 512, qptr[b + 1]))
            q = s["q"][rows].double().view(-1, hk, hq // hk, D)
            logit = torch.einsum("thgd,nhd->thgn", q, kv[0]) / D ** 0.5
            if case["causal"]:
                place = torch.arange(n, device="cuda")[None, :] > torch.arange(n - m + at, n - m + at + q.shape[0], device="cuda")[:, None]
                logit = logit.masked_fill(place[:, None, None, :], -math.inf)
            lse[rows] = torch.logsumexp(logit, -1).reshape(-1, hq)
            out[rows] = torch.einsum("thgn,nhd->thgd", torch.softmax(logit, -1), kv[1]).reshape(-1, hq, D)
    return {"out": out, "lse": lse}
