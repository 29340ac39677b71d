"""8-bit caches of values of all sizes, appended as bf16, some of them beyond f16's range, read by queries of f16: as exact as stated at each test."""

import math

import pytest
import torch

from tests._attention import attend64, half_step, visible, weight64
from tests._cache8 import CODES, TOP, empty_cache, take, values
from tests.test_gpu_cache8_calls import gen, ints

pytestmark = pytest.mark.gpu
LARGE = [65280.0, 65536.0, 2.0 ** 20, 1e9, 1e15, 2.0 ** 120]
H, D, N = 2, 128, 300


def _assert_wide(got, got_lse, q, k, v, seen, scale, more):
    """assert_attention where a row may pass the type's range: there it is infinite.  more: what else a result may be off by."""
    want, lse, tol, tol_lse = attend64(q, k, v, seen, scale)
    top = torch.finfo(q.dtype).max
    tol = tol + half_step(q.dtype) * (weight64(q, k, v, seen, scale) + want.abs()) + torch.finfo(q.dtype).smallest_normal + more
    got = got.double()
    assert not bool(torch.isnan(got).any())
    beyond, within = want.abs() - tol > top * (1 + half_step(q.dtype)), want.abs() + tol < top
    assert torch.equal(got[beyond], want[beyond].sign() * math.inf)
    assert bool(((got - want).abs() <= tol)[within].all()), f"off by {float(((got - want).abs() - tol)[within].max())}"
    assert bool(((got_lse.double() - lse).abs() <= tol_lse).all())


def _cache(gpu, code, large, tiny=40):
    """Operands of a sequence of N positions whose head 0 has a large value at 200 and head 1 one at 290, and its keys and values in 64 bits."""
    g = gen(7)
    kc, ks = empty_cache(24, 16, H, D, CODES[code])
    vc, vs = empty_cache(24, 16, H, D, CODES[code])
    pages = torch.randperm(24, generator=g, device="cuda").int()[:19].view(1, 19)
    k, v = (torch.randn((N, H, D), generator=g, device="cuda").bfloat16() for _ in range(2))
    k[200] *= 3  # of more and of less weight than others
    v[:tiny] *= 2.0 ** -60  # what is held against them is small when the large ones come
    v[200, 0, 5] = large
    v[290, 1, 7] = -large
    s = dict(k_scale=ks, v_scale=vs)
    gpu.kv_append(k, v, kc, vc, pages, ints(range(N)), seqs=ints([0] * N), **s)
    at = torch.arange(N, device="cuda")
    rows, at = pages[0].long()[at // 16], at % 16
    kq, vq = (values(take(c, rows, at), z[rows, :, at]) for c, z in ((kc, ks), (vc, vs)))
    return g, dict(k_cache=kc, v_cache=vc, pages=pages, **s), kq, vq


def _steps(gpu, code, large, dt, more):
    g, cache, k, v = _cache(gpu, code, large)
    q = torch.randn((1, 4, D), generator=g, device="cuda").to(dt)
    lse = torch.empty((1, 4), device="cuda")
    for m in (N, 290, 200):
        for prefix in (None, 2):
            call = dict(lengths=ints([m]), lse=lse, **cache)
            out = gpu.attend_decode(q, **call) if prefix is None else gpu.attend_decode_shared(q, prefix=cache["pages"][0, :prefix], **call)
            _assert_wide(out, lse, q, k[:m], v[:m], visible(1, m, True, "cuda"), D ** -0.5, m * more if m > 200 else 0.0)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("large", LARGE)
def test_steps_of_half_queries(gpu, code, large):
    """Probability times scale is held in two summands of f16 against the largest scale's power, 2^e: a key is off by 2^-25 of 2^(e - 14) times a code
    of up to `top`, by the smaller summand's rounding."""
    e = math.floor(math.log2(large / TOP[CODES[code]]))
    _steps(gpu, code, large, torch.float16, 2.0 ** -25 * 2.0 ** (e - 14) * TOP[CODES[code]])


@pytest.mark.parametrize("code", CODES)
def test_steps_of_scales_further_apart_than_exponents(gpu, code):
    """Values of 2^-60, then one of 2^120 in a dimension that they have nothing in: f16 steps lose the small ones beside it, and make nothing of
    their own (here at most the weight of what is there)."""
    g, cache, k, v = _cache(gpu, code, 2.0 ** 120, tiny=128)
    q = torch.randn((1, 4, D), generator=g, device="cuda").half()
    for prefix in (None, 2):
        call = dict(lengths=ints([N]), **cache)
        out = gpu.attend_decode(q, **call) if prefix is None else gpu.attend_decode_shared(q, prefix=cache["pages"][0, :prefix], **call)
        size = weight64(q, k, v.clamp(-8, 8), visible(1, N, True, "cuda"), D ** -0.5)
        others = torch.arange(D, device="cuda") != 5
        assert bool((out[:, :2].double().abs() <= 1.01 * size[:, :2])[..., others].all())
        assert bool((out[:, :2, 5] == math.inf).all())
