"""8-bit caches of values of all sizes, appended as bf16, read by queries of both types.  To f16 queries a row whose largest f16 cannot hold is a
NaN, as a row with an infinity is: who sees it gets one, and nobody else; bf16 queries read all of them."""

import math

import pytest
import torch

from tests._attention import assert_attention, visible
from tests._cache8 import CODES, empty_cache, take, values
from tests.test_gpu_cache8_calls import gen, ints

pytestmark = pytest.mark.gpu
H, D, N = 2, 128, 300


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tiny", [40, 128])  # what is held against small values when the large ones come
@pytest.mark.parametrize("large", [65280.0, 65536.0, 2.0 ** 20, 1e9, 1e15, 2.0 ** 120])  # 65280: bf16's last that f16 can hold
def test_values_of_all_sizes(gpu, code, dt, large, tiny):
    g = gen(7)
    kc, ks = empty_cache(24, 16, H, D, CODES[code])
    vc, vs = empty_cache(24, 16, H, D, CODES[code])
    pages = torch.randperm(24, generator=g, device="cuda").int()[:19].view(1, 19)
    k, v = (torch.randn((N, H, D), generator=g, device="cuda").bfloat16() for _ in range(2))
    k[200] *= 3  # of more and of less weight than others
    v[:tiny] *= 2.0 ** -60
    v[200, 0, 5] = large
    v[290, 1, 7] = -large
    cache = dict(k_cache=kc, v_cache=vc, pages=pages, k_scale=ks, v_scale=vs)
    gpu.kv_append(k, v, positions=ints(range(N)), seqs=ints([0] * N), **cache)
    at = torch.arange(N, device="cuda")
    rows, at = pages[0].long()[at // 16], at % 16
    k, v = (values(take(c, rows, at), z[rows, :, at]) for c, z in ((kc, ks), (vc, vs)))
    if dt == torch.float16:
        v[v.abs().amax(-1) >= 65520] = math.nan
        assert bool(torch.isnan(v).any()) == (large > 65280)
    q = torch.randn((150, 4, D), generator=g, device="cuda").to(dt)
    lse = torch.empty((150, 4), device="cuda")
    out = gpu.attend_prompt_paged(q, lengths=ints([N]), starts=ints([0, 150]), lse=lse, **cache)
    seen = visible(150, N, True, "cuda")
    for h in (0, 1):  # a head's value is no other's
        of = slice(2 * h, 2 * h + 2)
        assert_attention(out[:, of], lse[:, of], q[:, of], k[:, h:h + 1], v[:, h:h + 1], seen, D ** -0.5)
    for m in (N, 290, 200):
        for prefix in (None, 2):
            call = dict(lengths=ints([m]), lse=lse[:1], **cache)
            out = gpu.attend_decode(q[:1], **call) if prefix is None else gpu.attend_decode_shared(q[:1], prefix=pages[0, :prefix], **call)
            for h in (0, 1):
                of = slice(2 * h, 2 * h + 2)
                assert_attention(out[:, of], lse[:1, of], q[:1, of], k[:m, h:h + 1], v[:m, h:h + 1], visible(1, m, True, "cuda"), D ** -0.5)


@pytest.mark.parametrize("code", CODES)
def test_a_large_value_in_a_long_shared_prefix(gpu, code):
    """The launches of a prefix's own: 70 sequences, of which the short ones do not see it."""
    g, B, P = gen(8), 70, 2048
    kc, ks = empty_cache(P // 16 + B, 16, H, D, CODES[code])
    vc, vs = empty_cache(P // 16 + B, 16, H, D, CODES[code])
    prefix = torch.randperm(P // 16, generator=g, device="cuda").int()
    pages = torch.cat((prefix.expand(B, -1), P // 16 + torch.arange(B, dtype=torch.int32, device="cuda")[:, None]), 1)
    k, v = (torch.randn((P, H, D), generator=g, device="cuda").bfloat16() for _ in range(2))
    v[1500, 1, 3] = 1e6
    cache = dict(k_cache=kc, v_cache=vc, pages=pages, k_scale=ks, v_scale=vs)
    gpu.kv_append(k, v, positions=ints(range(P)), seqs=ints([0] * P), **cache)
    at = torch.arange(P, device="cuda")
    rows, at = prefix.long()[at // 16], at % 16
    k, v = (values(take(c, rows, at), z[rows, :, at]) for c, z in ((kc, ks), (vc, vs)))
    v[1500, 1] = math.nan
    lengths = [1501 if b % 2 else 1500 for b in range(B)]
    q = torch.randn((B, 4, D), generator=g, device="cuda").half()
    lse = torch.empty((B, 4), device="cuda")
    out = gpu.attend_decode_shared(q, prefix=prefix, lengths=ints(lengths), lse=lse, **cache)
    for b in (0, 1, 68, 69):
        m = lengths[b]
        for h in (0, 1):
            of = slice(2 * h, 2 * h + 2)
            assert_attention(out[b:b + 1, of], lse[b:b + 1, of], q[b:b + 1, of], k[:m, h:h + 1], v[:m, h:h + 1], visible(1, m, True, "cuda"), D ** -0.5)
