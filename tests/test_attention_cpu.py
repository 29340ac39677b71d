"""The attention entry points without a GPU: argument checks of the C ABI, sizes, and what the Python calls refuse.

Only calls that return before any HIP runtime call are made here.
"""

import ctypes
import os
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def L():
    from latent_amd import _lib

    return _lib


BUF = np.zeros(4096, np.uint8)
P = BUF.ctypes.data + (-BUF.ctypes.data) % 16  # never read: every call returns before a launch


def _cache(L, **kw):
    f = dict(k=P, v=P, pages=P, n_pages=10, page_size=16, n_seq=4, max_pages=8, pages_stride=8, k_page_stride=16 * 128,
             k_row_stride=128, k_head_stride=64, v_page_stride=16 * 128, v_row_stride=128, v_head_stride=64)
    return L.LatentKvCache(**{**f, **kw})


def _append(L, cache=None, **kw):
    f = dict(cache=cache or _cache(L), q=P, q_out=P, k=P, v=P, q_token_stride=256, q_head_stride=64, q_out_token_stride=256,
             q_out_head_stride=64, k_token_stride=128, k_head_stride=64, v_token_stride=128, v_head_stride=64, positions=P,
             seqs=P, rope=P, rope_rows=100, rot_dim=64, n_tokens=4, n_head=4, n_kv_head=2, head_dim=64, dtype=L.LATENT_BF16,
             rope_kind=L.LATENT_ROPE_HALF)
    return L.LatentKvAppendArgs(**{**f, **kw})


def _decode(L, cache=None, **kw):
    f = dict(cache=cache or _cache(L, max_pages=400, pages_stride=400), q=P, out=P, lengths=P, q_token_stride=256, q_head_stride=64,
             out_token_stride=256, out_head_stride=64, n_head=4, n_kv_head=2, head_dim=64, dtype=L.LATENT_F16, scale=0.125)
    return L.LatentAttnDecodeArgs(**{**f, **kw})


def _prompt(L, cache=None, **kw):
    f = dict(cache=cache or _cache(L), q=P, out=P, k=P, v=P, starts=P, k_starts=P, lengths=P, q_token_stride=256, q_head_stride=64,
             out_token_stride=256, out_head_stride=64, k_token_stride=128, k_head_stride=64, v_token_stride=128,
             v_head_stride=64, n_tokens=20, n_keys=20, n_head=4, n_kv_head=2, head_dim=64, dtype=L.LATENT_F16, causal=1, scale=0.125)
    return L.LatentAttnPromptArgs(**{**f, **kw})


SHARED = [
    (dict(n_head=3), "INVALID"), (dict(n_kv_head=0), "INVALID"), (dict(head_dim=0), "INVALID"), (dict(head_dim=60), "UNSUPPORTED"),
    (dict(head_dim=264), "UNSUPPORTED"), (dict(dtype=0), "INVALID"), (dict(dtype=3), "INVALID"), (dict(n_head=-2), "INVALID"),
    (dict(q_token_stride=250), "UNSUPPORTED"), (dict(q_head_stride=-64), "UNSUPPORTED"), (dict(q=P + 8), "UNSUPPORTED"),
]
CACHE = [
    (dict(page_size=0), "INVALID"), (dict(n_pages=-1), "INVALID"), (dict(max_pages=-1), "INVALID"), (dict(n_seq=-1), "INVALID"),
    (dict(pages_stride=7), "INVALID"), (dict(k_row_stride=132), "UNSUPPORTED"), (dict(v_page_stride=-8), "UNSUPPORTED"),
    (dict(k=P + 2), "UNSUPPORTED"), (dict(page_size=1 << 30, max_pages=8), "UNSUPPORTED"), (dict(n_seq=1 << 21), "UNSUPPORTED"),
]


def _expect(L, call, status):
    assert call == getattr(L, "LATENT_E_" + status)


@pytest.mark.parametrize("change,status", SHARED + [
    (dict(n_tokens=-1), "INVALID"), (dict(rot_dim=63), "INVALID"), (dict(rot_dim=66), "INVALID"), (dict(rot_dim=0), "INVALID"),
    (dict(rope_kind=2), "INVALID"), (dict(k=None), "INVALID"), (dict(v=None), "INVALID"), (dict(positions=None), "INVALID"),
    (dict(q_out=None), "INVALID"), (dict(rope=P + 4), "UNSUPPORTED"), (dict(q_out_token_stride=0), "INVALID"),
    (dict(n_tokens=1 << 25), "UNSUPPORTED"), (dict(n_tokens=1 << 24, head_dim=256), "UNSUPPORTED"),
])
def test_append_argument_checks(L, change, status):
    _expect(L, L.lib.latent_kv_append(ctypes.byref(_append(L, **change)), None), status)


@pytest.mark.parametrize("change,status", CACHE + [(dict(k_head_stride=0), "INVALID"), (dict(v_row_stride=0), "INVALID"),
                                                   (dict(k=None), "INVALID"), (dict(pages=None), "INVALID")])
def test_append_cache_checks(L, change, status):
    _expect(L, L.lib.latent_kv_append(ctypes.byref(_append(L, cache=_cache(L, **change))), None), status)


@pytest.mark.parametrize("change,status", SHARED + [
    (dict(scale=0.0), "INVALID"), (dict(scale=-1.0), "INVALID"), (dict(scale=float("nan")), "INVALID"),
    (dict(scale=float("inf")), "INVALID"), (dict(lengths=None), "INVALID"), (dict(out=None), "INVALID"), (dict(n_head=0), "INVALID"),
    (dict(out_head_stride=0), "INVALID"), ({}, "WORKSPACE"), (dict(workspace=P, workspace_bytes=64), "WORKSPACE"),
    (dict(workspace=P + 8, workspace_bytes=1 << 30), "UNSUPPORTED"),
])
def test_decode_argument_checks(L, change, status):
    _expect(L, L.lib.latent_attn_decode(ctypes.byref(_decode(L, **change)), None), status)


@pytest.mark.parametrize("change,status", CACHE + [(dict(pages=None), "INVALID"), (dict(v=None), "INVALID"),
                                                   (dict(n_seq=1 << 20, max_pages=1 << 20), "UNSUPPORTED")])
def test_decode_cache_checks(L, change, status):
    big = dict(max_pages=400, pages_stride=1 << 20) if "pages_stride" not in change else dict(max_pages=400)
    _expect(L, L.lib.latent_attn_decode(ctypes.byref(_decode(L, cache=_cache(L, **{**big, **change}))), None), status)


@pytest.mark.parametrize("change,status", SHARED + [
    (dict(scale=0.0), "INVALID"), (dict(n_tokens=-1), "INVALID"), (dict(n_keys=-1), "INVALID"), (dict(starts=None), "INVALID"),
    (dict(k_starts=None), "INVALID"), (dict(v=None), "INVALID"), (dict(v=P + 4), "UNSUPPORTED"), (dict(k_token_stride=4), "UNSUPPORTED"),
    (dict(k_token_stride=(1 << 24) + 8), "UNSUPPORTED"), (dict(n_tokens=1 << 29), "UNSUPPORTED"), (dict(out_token_stride=0), "INVALID"),
    (dict(k=None, n_keys=0, lengths=None), "INVALID"), (dict(k=None), "INVALID"),
])
def test_prompt_argument_checks(L, change, status):
    _expect(L, L.lib.latent_attn_prompt(ctypes.byref(_prompt(L, **change)), None), status)


@pytest.mark.parametrize("change,status", CACHE + [(dict(pages=None), "INVALID"), (dict(v=None), "INVALID")])
def test_prompt_cache_checks(L, change, status):
    _expect(L, L.lib.latent_attn_prompt(ctypes.byref(_prompt(L, cache=_cache(L, **change), k=None, n_keys=0)), None), status)


def test_calls_of_no_size_succeed(L):
    assert L.lib.latent_kv_append(ctypes.byref(_append(L, n_tokens=0, k=None)), None) == L.LATENT_OK
    assert L.lib.latent_attn_decode(ctypes.byref(_decode(L, cache=_cache(L, n_seq=0), q=None)), None) == L.LATENT_OK
    assert L.lib.latent_attn_prompt(ctypes.byref(_prompt(L, n_tokens=0, q=None)), None) == L.LATENT_OK
    for f in ("latent_kv_append", "latent_attn_decode", "latent_attn_prompt"):
        assert getattr(L.lib, f)(None, None) == L.LATENT_E_INVALID


def test_decode_workspace_grows_to_a_bound(L):
    """Two parts a workgroup, whatever the sequences: B = 4 or 400 of 64 heads of 128 need less than 40 MiB."""
    last = 0
    n = ctypes.c_size_t()
    for seqs, pages in ((1, 40), (4, 400), (400, 4000)):
        a = _decode(L, cache=_cache(L, n_seq=seqs, max_pages=pages, pages_stride=pages), n_head=64, n_kv_head=8, head_dim=128)
        assert L.lib.latent_attn_decode_workspace_size(ctypes.byref(a), ctypes.byref(n)) == L.LATENT_OK
        assert last <= n.value < 40 << 20
        last = n.value
    short = _decode(L, cache=_cache(L, n_seq=400, max_pages=8))
    assert L.lib.latent_attn_decode_workspace_size(ctypes.byref(short), ctypes.byref(n)) == L.LATENT_OK and n.value == 0
    import latent_amd

    assert latent_amd.attend_decode_workspace_size(400, 64, 8, 128, 4000, 16) == last
    with pytest.raises(latent_amd.LatentError):
        latent_amd.attend_decode_workspace_size(1, 3, 2, 128, 40, 16)


def test_prompt_workspace_follows_the_call(L):
    """A part is 128 rows of D rounded up to 64, 128 or 256 in fp32, and 16 bytes for each of 256 threads: 68 KB at D = 128.  A call
    has no more of them than row tiles times chunks of 256 keys, nor than 1280."""
    import latent_amd as la

    size = la.attend_prompt_workspace_size
    part = 128 * 128 * 4 + 256 * 16
    assert 0 < size(600, 1, 1, 1, 128, n_keys=600) <= 5 * 3 * part
    assert 0 < size(5, 1, 8, 8, 64, max_pages=40, page_size=32) <= 8 * 5 * part  # 8 row tiles, 1280 keys
    assert 0 < size(600, 1, 1, 1, 256, n_keys=600) <= 5 * 3 * 2 * part
    last = 0
    for keys in (600, 6000, 60000, 600000):
        n = size(64, 4, 8, 2, 128, max_pages=keys // 100, page_size=100)
        assert last <= n <= 1280 * part
        last = n
    assert last == 1280 * part  # long keys: the most there are


# ---- the Python calls -----------------------------------------------------------
def _t(*shape, dt=torch.bfloat16):
    return torch.zeros(shape, dtype=dt)


def _calls():
    import latent_amd as la

    kc, pages, ints = _t(4, 8, 2, 64), torch.zeros((3, 2), dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    return {
        "kv_append": lambda q: la.kv_append(q, q, kc, kc, pages, ints),
        "attend_decode": lambda q: la.attend_decode(q, kc, kc, pages, ints),
        "attend_prompt": lambda q: la.attend_prompt(q, q, q, ints),
        "attend_prompt_paged": lambda q: la.attend_prompt_paged(q, kc, kc, pages, ints, ints),
    }


@pytest.mark.parametrize("name", ["kv_append", "attend_decode", "attend_prompt", "attend_prompt_paged"])
def test_cpu_tensors_are_refused(name):
    with pytest.raises(ValueError, match="CUDA"):
        _calls()[name](_t(3, 2, 64))


@pytest.mark.parametrize("name", ["kv_append", "attend_decode", "attend_prompt", "attend_prompt_paged"])
def test_what_is_no_tensor_is_refused(name):
    for bad in (None, 3, np.zeros((3, 2, 64), np.float16)):
        with pytest.raises(TypeError, match="must be a tensor"):
            _calls()[name](bad)


def test_rope_table_on_the_cpu():
    import latent_amd as la

    t = la.rope_table(50, 8, base=100.0, device="cpu")
    assert t.shape == (50, 2, 4) and t.dtype == torch.float32 and t.is_contiguous()
    for p in (0, 1, 49):
        for i in range(4):
            angle = p * 100.0 ** (-2 * i / 8)
            assert t[p, 0, i] == np.float32(np.cos(angle)) and t[p, 1, i] == np.float32(np.sin(angle))
    for bad in ((5, 7), (5, 0), (-1, 8)):
        with pytest.raises(ValueError):
            la.rope_table(*bad, device="cpu")


# ---- without the binding --------------------------------------------------------
def test_the_package_imports_without_the_binding():
    """Only the attention calls need _attend.so; where it is missing or does not load, they say so."""
    code = """
import sys
sys.modules["latent_amd._attend"] = None
import torch, latent_amd as la, latent_amd.gguf
assert la.moe_forward and la.Router and la.library_version() >= 100
assert la.attend_decode_workspace_size(1, 4, 2, 64, 400, 16) > 0
t = torch.zeros((1, 1, 8))
for call in (lambda: la.kv_append(t, t, t, t, t, t), lambda: la.attend_decode(t, t, t, t, t), lambda: la.attend_prompt(t, t, t, t),
             lambda: la.attend_prompt_paged(t, t, t, t, t, t)):
    try:
        call()
    except ImportError as e:
        assert "_attend.so" in str(e) and "build.py" in str(e)
    else:
        raise AssertionError("no error")
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.parametrize("why", ["no torch", "no compiler", "an error"])
def test_the_library_is_built_whatever_becomes_of_the_binding(tmp_path, monkeypatch, why):
    from latent_amd import build as b

    if not os.path.exists(b.hipcc()):
        pytest.skip("hipcc not found")
    for name, value in (("PKG", tmp_path), ("LIB", tmp_path / "lib.so"), ("BINDING", tmp_path / "binding.so"), ("SOURCES", ["noalloc.hip"])):
        monkeypatch.setattr(b, name, value)
    if why == "no torch":
        monkeypatch.setattr(b.importlib.util, "find_spec", lambda name: None)
        b.build()
    else:
        monkeypatch.setenv("CXX", "/nowhere/g++" if why == "no compiler" else "false")
        with pytest.raises(RuntimeError, match="_attend|binding"):
            b.build()
    assert b.LIB.exists() and not b.BINDING.exists()
