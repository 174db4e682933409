"""CPU checks of the prefill, page copy and draft verification entry points:
struct layouts, argument checks by status code before the device is touched,
and refusals of CPU tensors and of host lists that would race."""
import ctypes
import os
import subprocess

import pytest
import torch

from ecahlang_b200 import _abi, drafts, paged
from ecahlang_b200.build import ROOT, build
from test_operators_cpu import BAD_CACHES, _cache, _set


@pytest.fixture(scope="module")
def L():
    build()
    return _abi.lib()


@pytest.mark.parametrize("mirror,cname", [(_abi.PrefillArgs, "ecah_prefill_args"), (_abi.CopyArgs, "ecah_copy_args"),
                                          (_abi.VerifyArgs, "ecah_verify_args")])
def test_struct_layout_matches_header(tmp_path, mirror, cname):
    fields = [n for n, _ in mirror._fields_]
    src = tmp_path / "off.c"
    src.write_text("#include <stdio.h>\n#include <stddef.h>\n#include \"ecah_sampler.h\"\nint main(){"
                   + "".join(f'printf("%zu\\n", offsetof({cname}, {f}));' for f in fields)
                   + f'printf("%zu\\n", sizeof({cname}));return 0;}}')
    exe = tmp_path / "off"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [getattr(mirror, f).offset for f in fields] + [ctypes.sizeof(mirror)]


def test_prefill_rejects_bad_arguments_without_a_device(L):
    def a(cache=None, **kw):
        base = dict(abi_version=_abi.ABI_VERSION, dtype=1, tokens=5, num_qo_heads=8, sm_scale=0.1, causal=1, q=64, out=64,
                    qo_indptr=64, kv_last_page_len=64, cache=_cache(**(cache or {})))
        return _set(_abi.PrefillArgs(), {**base, **kw})
    f = L.ecah_paged_prefill
    assert f(None, None) == 1
    assert f(a(abi_version=9), None) == 6
    assert f(a(dtype=2), None) == 2
    for cache, status in BAD_CACHES:
        assert f(a(cache=cache), None) == status, cache
    assert f(a(tokens=-1), None) == 3
    assert f(a(num_qo_heads=9), None) == 3
    assert f(a(num_qo_heads=0), None) == 3
    for scale in (0.0, -1.0, float("nan")):
        assert f(a(sm_scale=scale), None) == 3
    assert f(a(q_token_stride=4), None) == 3
    assert f(a(out_head_stride=-8), None) == 3
    assert f(a(tokens=0), None) == 0
    assert f(a(cache=dict(batch=0)), None) == 0
    assert f(a(q=None), None) == 1
    assert f(a(qo_indptr=None), None) == 1
    assert f(a(kv_last_page_len=None), None) == 1
    assert f(a(out=72), None) == 3
    assert f(a(), None) == 4                                  # no workspace
    for off in (1, 2, 4, 8, 24):
        assert f(a(workspace=4096 + off, workspace_bytes=1 << 30), None) == 4
    assert L.ecah_paged_prefill_workspace_bytes(100) == 0


def test_copy_rejects_bad_arguments_without_a_device(L):
    ptrs = (ctypes.c_void_p * 3)(64, 128, 192)
    null = (ctypes.c_void_p * 3)(64, None, 192)
    off = (ctypes.c_void_p * 3)(64, 72, 192)

    def a(**kw):
        base = dict(abi_version=_abi.ABI_VERSION, kv_dtype=1, num_pages=4, page_size=16, num_kv_heads=2, head_dim=64, layers=3,
                    pairs=2, k_page_stride=2048, k_slot_stride=128, k_head_stride=64, v_page_stride=2048, v_slot_stride=128,
                    v_head_stride=64, k_caches=ctypes.addressof(ptrs), v_caches=ctypes.addressof(ptrs), src=64, dst=64)
        return _set(_abi.CopyArgs(), {**base, **kw})
    f = L.ecah_paged_copy
    assert f(None, None) == 1
    assert f(a(abi_version=1), None) == 6
    assert f(a(kv_dtype=2), None) == 2
    for bad in (dict(num_pages=-1), dict(page_size=0), dict(num_kv_heads=0), dict(head_dim=80), dict(layers=-1), dict(pairs=-1),
                dict(k_slot_stride=100), dict(v_head_stride=-64), dict(kv_dtype=_abi.KV_E4M3, k_head_stride=72)):
        assert f(a(**bad), None) == 3, bad
    for none in (dict(layers=0), dict(pairs=0), dict(num_pages=0)):
        assert f(a(**none), None) == 0, none
    for bad in (dict(src=None), dict(dst=None), dict(k_caches=None), dict(v_caches=ctypes.addressof(null)),
                dict(kv_dtype=_abi.KV_E4M3), dict(kv_dtype=_abi.KV_E4M3, k_scales=ctypes.addressof(null), v_scales=ctypes.addressof(ptrs))):
        assert f(a(**bad), None) == 1, bad
    assert f(a(k_caches=ctypes.addressof(off)), None) == 3
    assert f(a(page_size=1 << 24, num_kv_heads=1 << 10), None) == 3      # more chunks a page than 32 bits count


def test_verify_rejects_bad_arguments_without_a_device(L):
    def a(**kw):
        base = dict(abi_version=_abi.ABI_VERSION, dtype=2, batch=2, drafts=3, vocab=100, target=64, draft_ids=64, uniforms=64,
                    tokens=64, accepted=64)
        return _set(_abi.VerifyArgs(), {**base, **kw})
    f = L.ecah_verify_drafts
    assert f(None, None) == 1
    assert f(a(abi_version=1), None) == 6
    assert f(a(dtype=3), None) == 2
    for bad in (dict(batch=-1), dict(batch=65536), dict(drafts=-1), dict(drafts=2 ** 31 - 1), dict(vocab=0), dict(vocab=2 ** 31 - 1),
                dict(target_row_stride=-1), dict(draft_batch_stride=-4)):
        assert f(a(**bad), None) == 3, bad
    assert f(a(batch=0), None) == 0
    for bad in ("target", "uniforms", "tokens", "accepted", "draft_ids"):
        assert f(a(**{bad: None}), None) == 1, bad
    assert f(a(), None) == 4
    need = L.ecah_verify_drafts_workspace_bytes(2)
    assert f(a(workspace=4096, workspace_bytes=need - 1), None) == 4
    for off in (1, 4, 8):
        assert f(a(workspace=4096 + off, workspace_bytes=need), None) == 4
    assert L.ecah_verify_drafts_workspace_bytes(-1) == 0


def test_cpu_tensors_are_rejected():
    ids = torch.zeros(2, dtype=torch.int32)
    ws = torch.zeros(256, dtype=torch.uint8)
    q = torch.zeros(2, 1, 64, dtype=torch.float16)
    c = torch.zeros(2, 16, 1, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged.prefill(q, ids, ids, ids[:1], ids[:1], c, c, ws)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged.copy_pages([0], [1], [(c, c, None, None)])
    with pytest.raises(RuntimeError, match="CUDA"):
        drafts.verify(torch.zeros(1, 2, 8), ids[:1].view(1, 1), torch.zeros(1, 2), ws)


@pytest.mark.parametrize("src,dst,tokens,why", [
    ([0, 1], [2], None, "2 source and 1 destination"), ([0, 1], [2, 2], None, "must differ"), ([0, 1], [2, 0], None, "must differ"),
    ([0], [0], None, "must differ"), ([0], [4], None, "page outside"), ([-1], [2], None, "page outside"),
    ([0], [2], [17], "tokens must be"), ([0], [2], [-1], "tokens must be"), ([0], [2], [], "tokens must be")])
def test_page_lists_that_would_race_or_overrun_are_refused(src, dst, tokens, why):
    c = torch.zeros(4, 16, 1, 64, dtype=torch.float16)
    with pytest.raises((RuntimeError, IndexError), match=why):
        paged.copy_pages(src, dst, [(c, c, None, None)], tokens=tokens)


def test_no_layers_is_no_work():
    paged.copy_pages([0], [1], [])
