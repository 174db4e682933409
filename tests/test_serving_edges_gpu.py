"""Edges of the serving operators on the GPU against float64: what a wrong
answer hides behind in ordinary inputs."""
import math

import pytest
import torch

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
