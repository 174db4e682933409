"""CPU checks of the log-probability and paged-cache entry points: struct
layouts, argument checks by status code before the device is touched, and
refusals of CPU tensors."""
import ctypes
import os
import subprocess

import pytest
import torch

from ecahlang_b200 import _abi, logprobs, paged
from ecahlang_b200.build import ROOT, build


@pytest.fixture(scope="module")
def L():
    build()
    return _abi.lib()


@pytest.mark.parametrize("mirror,cname", [(_abi.LogprobArgs, "ecah_logprob_args"), (_abi.KVCache, "ecah_kv_cache"),
                                          (_abi.AppendArgs, "ecah_append_args"), (_abi.DecodeArgs, "ecah_decode_args")])
def test_struct_layout_matches_header(tmp_path, mirror, cname):
    fields = [n for n, _ in mirror._fields_]
    src = tmp_path / "off.c"
    src.write_text("#include <stdio.h>\n#include <stddef.h>\n#include \"ecah_sampler.h\"\nint main(){"
                   + "".join(f'printf("%zu\\n", offsetof({cname}, {f}));' for f in fields)
                   + f'printf("%zu\\n", sizeof({cname}));'
                   + 'printf("%d %d\\n", ECAH_KV_E4M3, ECAH_MAX_TOP_N);return 0;}')
    exe = tmp_path / "off"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [getattr(mirror, f).offset for f in fields] + [ctypes.sizeof(mirror), _abi.KV_E4M3, _abi.MAX_TOP_N]


def _set(a, kw):
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


def test_logprobs_rejects_bad_arguments_without_a_device(L):
    def a(**kw):
        return _set(_abi.LogprobArgs(abi_version=_abi.ABI_VERSION, dtype=0, rows=2, vocab=10, row_stride=10), kw)
    f = L.ecah_token_logprobs
    assert f(None, None) == 1
    assert f(a(abi_version=1), None) == 6
    assert f(a(dtype=3), None) == 2
    assert f(a(vocab=0), None) == 3
    assert f(a(row_stride=9), None) == 3
    assert f(a(top_n=33), None) == 3
    assert f(a(tokens_per_row=-1), None) == 3
    assert f(a(rows=-1), None) == 3
    assert f(a(vocab=2 ** 31 - 1, row_stride=2 ** 31), None) == 3
    assert f(a(row_index=16), None) == 3                      # no rows to gather from
    assert f(a(rows=0), None) == 0
    assert f(a(), None) == 1                                  # no logits
    assert f(a(logits=16, tokens_per_row=1), None) == 1       # no token ids
    assert f(a(logits=16, top_n=1), None) == 1                # no outputs
    assert f(a(logits=16), None) == 4                         # no workspace


def _cache(**kw):
    c = _abi.KVCache(kv_dtype=1, num_pages=4, page_size=16, num_kv_heads=2, head_dim=64, batch=2, k_cache=64, v_cache=64,
                     k_page_stride=2048, k_slot_stride=128, k_head_stride=64, v_page_stride=2048, v_slot_stride=128,
                     v_head_stride=64, kv_indptr=64, kv_indices=64, num_indices=4)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


BAD_CACHES = [(dict(kv_dtype=0), 2), (dict(kv_dtype=2), 2), (dict(head_dim=80), 3), (dict(page_size=0), 3), (dict(num_kv_heads=0), 3),
              (dict(num_pages=-1), 3), (dict(batch=-1), 3), (dict(num_indices=-1), 3), (dict(kv_indptr=None), 1),
              (dict(kv_indices=None), 1), (dict(k_cache=None), 1), (dict(k_slot_stride=100), 3), (dict(v_head_stride=-64), 3),
              (dict(k_cache=24), 3), (dict(kv_dtype=_abi.KV_E4M3), 1),
              (dict(kv_dtype=_abi.KV_E4M3, k_scale=64, v_scale=64, k_head_stride=72), 3)]


def test_append_rejects_bad_arguments_without_a_device(L):
    def a(cache=None, **kw):
        base = dict(abi_version=_abi.ABI_VERSION, dtype=1, tokens=3, num_qo_heads=8, q=64, k=64, v=64, q_out=64, positions=64,
                    batch_index=64, eps=1e-6, cache=_cache(**(cache or {})))
        return _set(_abi.AppendArgs(), {**base, **kw})
    f = L.ecah_paged_append
    assert f(None, None) == 1
    assert f(a(abi_version=9), None) == 6
    assert f(a(dtype=2), None) == 2
    for cache, status in BAD_CACHES:
        assert f(a(cache=cache), None) == status, cache
    assert f(a(tokens=-1), None) == 3
    assert f(a(cos_sin=64), None) == 3                        # a table without rows
    assert f(a(q_token_stride=4), None) == 3
    assert f(a(tokens=0), None) == 0
    assert f(a(k=None), None) == 1
    assert f(a(positions=None), None) == 1
    assert f(a(q_out=None), None) == 1
    assert f(a(q=None), None) == 3                            # heads without queries
    assert f(a(num_qo_heads=0), None) == 3
    assert f(a(v=72), None) == 3                              # not on a 16-byte boundary


def test_decode_rejects_bad_arguments_without_a_device(L):
    def a(cache=None, **kw):
        base = dict(abi_version=_abi.ABI_VERSION, dtype=1, num_qo_heads=8, sm_scale=0.1, q=64, out=64, kv_last_page_len=64,
                    cache=_cache(**(cache or {})))
        return _set(_abi.DecodeArgs(), {**base, **kw})
    f = L.ecah_paged_decode
    assert f(None, None) == 1
    assert f(a(abi_version=9), None) == 6
    assert f(a(dtype=2), None) == 2
    for cache, status in BAD_CACHES:
        assert f(a(cache=cache), None) == status, cache
    assert f(a(num_qo_heads=9), None) == 3
    assert f(a(num_qo_heads=0), None) == 3
    assert f(a(sm_scale=0.0), None) == 3
    assert f(a(sm_scale=float("nan")), None) == 3
    assert f(a(out_head_stride=4), None) == 3
    assert f(a(cache=dict(batch=0)), None) == 0
    assert f(a(q=None), None) == 1
    assert f(a(out=72), None) == 3
    assert f(a(), None) == 4                                  # no workspace
    assert L.ecah_paged_decode_workspace_bytes(4, 9, 2, 128) == 0
    assert L.ecah_paged_decode_workspace_bytes(4, 8, 2, 100) == 0


def test_cpu_tensors_are_rejected():
    x = torch.zeros(2, 8, dtype=torch.float16)
    ids = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        logprobs.launch(x, ids, torch.zeros(256, dtype=torch.uint8))
    k = torch.zeros(1, 1, 64, dtype=torch.float16)
    c = torch.zeros(2, 16, 1, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged.append(k, k, k, ids[:1], ids[:1], ids, ids[:1], c, c)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged.decode(k, ids, ids[:1], ids[:1], c, c, torch.zeros(256, dtype=torch.uint8))


def test_misaligned_workspaces_are_refused_without_a_device(L):
    """The kernels read and write their workspaces 16 bytes at a time."""
    lp = dict(abi_version=_abi.ABI_VERSION, dtype=0, rows=2, vocab=10, row_stride=10, logits=16, workspace_bytes=1 << 30)
    dec = dict(abi_version=_abi.ABI_VERSION, dtype=1, num_qo_heads=8, sm_scale=0.1, q=64, out=64, kv_last_page_len=64,
               cache=_cache(), workspace_bytes=1 << 30)
    for off in (1, 2, 4, 8, 24):
        assert L.ecah_token_logprobs(_set(_abi.LogprobArgs(), dict(lp, workspace=4096 + off)), None) == 4
        assert L.ecah_paged_decode(_set(_abi.DecodeArgs(), dict(dec, workspace=4096 + off)), None) == 4


def test_misaligned_sampler_workspaces_are_refused_without_a_device(L):
    """Counters are 32-bit; the row kernel's candidates 64-bit."""
    a = dict(abi_version=_abi.ABI_VERSION, dtype=0, batch=2, vocab=1000, row_stride=1000, logits=4096, temperature=4096,
             top_k=4096, top_p=4096, out=4096, uniforms=4096, workspace_bytes=1 << 30)
    for off in (1, 2, 4, 6):
        assert L.ecah_sampler_launch(_set(_abi.SamplerArgs(), dict(a, workspace=4096 + off)), None) == 4
    vp = dict(abi_version=_abi.ABI_VERSION, dtype=0, batch=1, vocab=1000, row_stride=1000, logits=4096, world=1,
              vocab_local=1000, cand_cap=64, temperature=4096, top_k=4096, top_p=4096, out=4096, uniforms=4096, all_cand=4096,
              all_count=4096, workspace_bytes=256)
    for off in (1, 2):
        assert L.ecah_vp_merge(_set(_abi.VPArgs(), dict(vp, workspace=4096 + off)), None) == 4


def test_manager_makes_no_workspace_inside_a_capture(monkeypatch):
    from ecahlang_b200.manager import SamplingManager
    m = SamplingManager(100, seq_lens=8, dtype=torch.float16, device="cpu", history_capacity=16)
    m.init_sampling_buffers(2)
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    x = torch.zeros(2, 100, dtype=torch.float16)
    for call in (lambda: m.sample(x), lambda: m.logprobs(x, None)):
        with pytest.raises(RuntimeError, match="inside a CUDA-graph capture"):
            call()


def test_manager_logprobs_checks_a_host_row_index():
    from ecahlang_b200.manager import SamplingManager
    m = SamplingManager(100, seq_lens=8, dtype=torch.float16, device="cpu", history_capacity=16)
    m.init_sampling_buffers(2)
    x = torch.zeros(5, 100, dtype=torch.float16)
    for bad in ([0, 5], [-1], torch.tensor([7]), range(4, 6)):
        with pytest.raises(IndexError, match="row_index"):
            m.logprobs(x, None, row_index=bad, tempered=True)


@pytest.mark.parametrize("dtype,kv,run", [(torch.float16, False, 16), (torch.bfloat16, False, 64),
                                          (torch.bfloat16, True, 16)])
def test_long_decode_tolerance_sees_a_lost_run_of_keys(dtype, kv, run):
    """Values of `run` neighbouring keys left out of the oracle's sum exceed the tolerance, wherever they lie."""
    from decode_util import long_cache, long_reference
    g = torch.Generator().manual_seed(1)
    n = 20000
    q = (torch.randn(4, 64, generator=g) * 1.5).to(dtype)
    cache = long_cache(n, 16, 2, 64, dtype, kv, g, "cpu")
    want, _, tol = long_reference(q, n, *cache, dtype)
    for at in (0, 7000, 12345, n - run):
        got, _, _ = long_reference(q, n, *cache, dtype, lost=slice(at, at + run))
        assert (((got - want).abs() / tol).amax(-1) > 1).all(), at
