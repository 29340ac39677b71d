"""The 8-bit caches', the shared prefix's and residual_norm's entry points without a GPU: argument checks of the C ABI, sizes, and
what the Python calls refuse.  Only calls that return before any HIP runtime call are made here."""

import ctypes

import pytest
import torch

from tests.test_attention_cpu import CACHE, P, SHARED, _append, _cache, _decode, _prompt


@pytest.fixture(scope="module")
def L():
    from latent_amd import _lib

    return _lib


def _scales(L, **kw):
    f = dict(k=P, v=P, k_page_stride=32, k_head_stride=16, v_page_stride=32, v_head_stride=16, code=L.LATENT_CODE_INT8)
    return L.LatentKvScales(**{**f, **kw})


def _read(L, cache=None, **kw):
    f = dict(cache=cache or _cache(L), k=P, v=P, k_token_stride=128, k_head_stride=64, v_token_stride=128, v_head_stride=64, positions=P,
             seqs=P, n_tokens=4, n_kv_head=2, head_dim=64, dtype=L.LATENT_BF16)
    return L.LatentKvReadArgs(**{**f, **kw})


def _shared(L, scales=None, n_prefix=3, prefix=P, cache=None, **kw):
    a = L.LatentAttnSharedArgs(decode=_decode(L, cache=cache, **kw), prefix=prefix, n_prefix=n_prefix)
    if scales is not None:
        a.scales = ctypes.pointer(scales)
    return a


def _norm(L, post=None, pre=None, **kw):
    f = dict(x=P, y=P, gate=P, x_out=P, n_out=P, x_stride=64, y_stride=64, gate_stride=0, x_out_stride=64, n_out_stride=64, n_tokens=3,
             n_embd=64, n_dtype=L.LATENT_BF16, scale=1.0,
             post=L.LatentNorm(**{**dict(kind=1, eps=1e-6, weight=P), **(post or {})}), pre=L.LatentNorm(**{**dict(kind=2, weight=P, bias=P), **(pre or {})}))
    return L.LatentResidualNormArgs(**{**f, **kw})


def _expect(L, got, status):
    assert got == (0 if status == "OK" else getattr(L, "LATENT_E_" + status))


CODES = [
    (dict(code=2), "INVALID"), (dict(code=-1), "INVALID"), (dict(k=P + 4), "UNSUPPORTED"), (dict(v=P + 8), "UNSUPPORTED"), (dict(k_page_stride=30), "UNSUPPORTED"),
    (dict(v_head_stride=-4), "UNSUPPORTED"), (dict(v_page_stride=(1 << 40) + 4), "UNSUPPORTED"),
]
CACHE8 = [(dict(page_size=12), "UNSUPPORTED"), (dict(k_row_stride=136), "UNSUPPORTED"), (dict(v_head_stride=72), "UNSUPPORTED")]


def _all(L):
    """Each entry point on 8-bit operands: f(scales, cache, **args)."""
    ref, lib = ctypes.byref, L.lib
    wide = lambda kw: _cache(L, **{**dict(max_pages=400, pages_stride=400), **kw})  # noqa: E731
    return {
        "append": lambda s, c, **kw: lib.latent_kv_append_q8(ref(_append(L, cache=_cache(L, **c), **kw)), ref(s), None),
        "read": lambda s, c, **kw: lib.latent_kv_read(ref(_read(L, cache=_cache(L, **c), **kw)), ref(s), None),
        "decode": lambda s, c, **kw: lib.latent_attn_decode_q8(ref(_decode(L, cache=wide(c), **kw)), ref(s), None),
        "prompt": lambda s, c, **kw: lib.latent_attn_prompt_q8(ref(_prompt(L, cache=_cache(L, **c), **{**dict(k=None, n_keys=0), **kw})), ref(s), None),
        "shared": lambda s, c, **kw: lib.latent_attn_decode_shared(ref(_shared(L, s, cache=wide(c), **kw)), None),
    }


@pytest.mark.parametrize("call", ["append", "read", "decode", "prompt", "shared"])
@pytest.mark.parametrize("change,status", CODES)
def test_scales_are_checked(L, call, change, status):
    _expect(L, _all(L)[call](_scales(L, **change), {}), status)


@pytest.mark.parametrize("call", ["append", "read", "decode", "prompt", "shared"])
@pytest.mark.parametrize("change,status", CACHE8 + [c for c in CACHE if "pages_stride" not in c[0]])
def test_caches_are_checked(L, call, change, status):
    _expect(L, _all(L)[call](_scales(L), change), status)


@pytest.mark.parametrize("call", ["append", "decode", "prompt", "shared"])
@pytest.mark.parametrize("change,status", SHARED + [(dict(head_dim=72), "UNSUPPORTED")])
def test_sizes_are_checked(L, call, change, status):
    _expect(L, _all(L)[call](_scales(L), {}, **change), status)


@pytest.mark.parametrize("call", ["append", "read", "decode", "prompt", "shared"])
def test_missing_scales(L, call):
    more = dict(workspace=P, workspace_bytes=1 << 40) if call in ("decode", "shared") else {}
    _expect(L, _all(L)[call](_scales(L, v=None), {}, **more), "INVALID")
    if call == "append":
        _expect(L, _all(L)[call](_scales(L, k_head_stride=0), {}), "INVALID")
        _expect(L, _all(L)[call](_scales(L, v_page_stride=0), {}), "INVALID")
    elif call != "read":
        f = {"decode": L.lib.latent_attn_decode_q8, "prompt": L.lib.latent_attn_prompt_q8}.get(call)
        if f:
            _expect(L, f(ctypes.byref(_decode(L) if call == "decode" else _prompt(L)), None, None), "INVALID")


@pytest.mark.parametrize("change,status", [
    (dict(n_tokens=-1), "INVALID"), (dict(n_tokens=1 << 25), "UNSUPPORTED"), (dict(n_kv_head=0), "INVALID"), (dict(head_dim=300), "UNSUPPORTED"),
    (dict(k=None), "INVALID"), (dict(positions=None), "INVALID"), (dict(v=P + 8), "UNSUPPORTED"), (dict(k_token_stride=4), "UNSUPPORTED"),
    (dict(v_head_stride=0), "INVALID"), (dict(dtype=0), "INVALID"), (dict(n_tokens=0, k=None), "OK")])
def test_read_argument_checks(L, change, status):
    for scales in (None, ctypes.byref(_scales(L))):
        _expect(L, L.lib.latent_kv_read(ctypes.byref(_read(L, **change)), scales, None), status)


def test_prompts_over_codes_take_no_packed_keys(L):
    _expect(L, L.lib.latent_attn_prompt_q8(ctypes.byref(_prompt(L)), ctypes.byref(_scales(L)), None), "INVALID")


@pytest.mark.parametrize("change,status", [
    (dict(n_prefix=-1), "INVALID"), (dict(n_prefix=401), "INVALID"), (dict(prefix=None), "INVALID"), (dict(lengths=None), "INVALID"), (dict(q=P + 8), "UNSUPPORTED"),
    ({}, "WORKSPACE"), (dict(workspace=P, workspace_bytes=64), "WORKSPACE"), (dict(workspace=P + 8, workspace_bytes=1 << 40), "UNSUPPORTED"),
    (dict(out_head_stride=0, workspace=P, workspace_bytes=1 << 40), "INVALID"), (dict(n_prefix=0), "WORKSPACE"), (dict(scale=0.0), "INVALID")])
def test_shared_prefix_argument_checks(L, change, status):
    for scales in (None, _scales(L)):
        _expect(L, L.lib.latent_attn_decode_shared(ctypes.byref(_shared(L, scales, **change)), None), status)


def test_shared_prefix_sizes(L):
    import latent_amd as la

    size = la.attend_decode_shared_workspace_size
    n = ctypes.c_size_t()
    for codes in (False, True):
        # Few sequences: a decode.  Many: the prefix's parts and those of the sequences' own keys.
        assert size(4, 8, 2, 64, 20, 16, 0, codes) >= la.attend_decode_workspace_size(4, 8, 2, 64, 20, 16, codes)
        assert size(64, 64, 8, 128, 300, 64, 250, codes) < 128 << 20
        assert size(1, 1, 1, 16, 1, 8, 1, codes) == 0
        assert size(5, 32, 8, 128, 300, 16, 256, codes) == la.attend_decode_workspace_size(5, 32, 8, 128, 300, 16, codes)
        assert size(60, 6, 2, 128, 40, 128, 32, codes) > la.attend_decode_workspace_size(60, 6, 2, 128, 40, 128, codes)
    with pytest.raises(la.LatentError):
        size(4, 8, 2, 64, 20, 16, 21)
    a = _shared(L, cache=_cache(L, n_seq=1 << 20, max_pages=1, pages_stride=1), n_head=1024, n_kv_head=1024, head_dim=256, n_prefix=1)
    _expect(L, L.lib.latent_attn_decode_shared_workspace_size(ctypes.byref(a), ctypes.byref(n)), "UNSUPPORTED")
    for f in (L.lib.latent_attn_decode_shared_workspace_size, L.lib.latent_attn_decode_q8_workspace_size):
        assert f(None, None) == L.LATENT_E_INVALID


@pytest.mark.parametrize("change,status", [
    (dict(n_tokens=-1), "INVALID"), (dict(n_embd=-1), "INVALID"), (dict(n_embd=32769), "UNSUPPORTED"), (dict(n_tokens=1 << 27), "UNSUPPORTED"), (dict(n_tokens=1 << 22, n_embd=16384), "UNSUPPORTED"), (dict(x=None), "INVALID"), (dict(x_dtype=3), "INVALID"),
    (dict(n_dtype=7), "INVALID"), (dict(gate_dtype=-1), "INVALID"), (dict(scale=float("nan")), "INVALID"), (dict(scale=float("inf")), "INVALID"), (dict(y=None), "INVALID"),
    (dict(y=None, gate=None), "INVALID"), (dict(n_out=None), "INVALID"), (dict(x_out_stride=63), "INVALID"), (dict(n_out_stride=0), "INVALID"), (dict(x_stride=-1), "UNSUPPORTED"),
    (dict(post=dict(kind=3)), "INVALID"), (dict(post=dict(kind=0)), "INVALID"), (dict(pre=dict(eps=-1.0)), "INVALID"), (dict(pre=dict(eps=float("nan"))), "INVALID"),
    (dict(pre=dict(dtype=5)), "INVALID"), (dict(n_tokens=0, x=None), "OK"), (dict(n_embd=0, x=None), "OK"), (dict(x_out=None, n_out=None, pre=dict(kind=0, weight=None, bias=None)), "OK")])
def test_norm_argument_checks(L, change, status):
    _expect(L, L.lib.latent_residual_norm(ctypes.byref(_norm(L, **change)), None), status)


def test_calls_without_arguments(L):
    for f in ("latent_kv_append_q8", "latent_kv_read", "latent_attn_decode_q8", "latent_attn_prompt_q8"):
        assert getattr(L.lib, f)(None, None, None) == L.LATENT_E_INVALID
    for f in ("latent_attn_decode_shared", "latent_residual_norm"):
        assert getattr(L.lib, f)(None, None) == L.LATENT_E_INVALID


# ---- the Python calls -----------------------------------------------------------
def test_cpu_tensors_and_what_is_no_tensor_are_refused():
    import latent_amd as la

    t, ints = torch.zeros((3, 2, 64), dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32)
    cache = torch.zeros((4, 8, 2, 64), dtype=torch.int8)
    scale, pages = la.kv_scales(cache), torch.zeros((3, 2), dtype=torch.int32)
    s = dict(k_scale=scale, v_scale=scale)
    for call in (lambda q: la.kv_append(q, q, cache, cache, pages, ints, **s), lambda q: la.attend_decode(q, cache, cache, pages, ints, **s),
                 lambda q: la.attend_prompt_paged(q, cache, cache, pages, ints, ints, **s), lambda q: la.attend_decode_shared(q, cache, cache, ints, pages, ints, **s)):
        with pytest.raises(ValueError, match="CUDA"):
            call(t)
        with pytest.raises(TypeError, match="must be a tensor"):
            call(None)
    with pytest.raises(ValueError, match="CUDA"):
        la.kv_read(cache, cache, pages, ints, dtype=torch.float16, **s)
    with pytest.raises(TypeError, match="must be a tensor"):
        la.kv_read(None, cache, pages, ints)
    with pytest.raises(TypeError):
        la.kv_read(cache, cache, pages, ints, dtype=torch.float32, **s)
    with pytest.raises(ValueError, match="CUDA"):
        la.residual_norm(torch.zeros((2, 8)), pre=la.Norm())
    for bad in (3, None):
        with pytest.raises(TypeError):
            la.residual_norm(bad)


def test_norms_and_scales_are_checked():
    import latent_amd as la

    for kw in (dict(kind="batch"), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf"))):
        with pytest.raises(ValueError):
            la.Norm(**kw)
    with pytest.raises(TypeError):
        la.residual_norm(torch.zeros((2, 8)), pre="rms")
    with pytest.raises(TypeError):
        la.residual_norm(torch.zeros((2, 8), dtype=torch.int32))
    with pytest.raises(ValueError):
        la.BlockNorm(gate=torch.zeros((2, 8)))
    for bad in (torch.zeros((2, 8, 1, 16)), torch.zeros((2, 8, 16), dtype=torch.int8)):
        with pytest.raises(TypeError):
            la.kv_scales(bad)
    assert la.kv_scales(torch.zeros((2, 8, 3, 16), dtype=torch.int8)).shape == (2, 3, 8)
