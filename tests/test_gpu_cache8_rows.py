"""8-bit rows that are not finite: who sees one gets a NaN, but its key counts in the log-sum-exp as any other."""

import math

import pytest
import torch

from tests._attention import assert_attention, visible
from tests._cache8 import CODES, paged8
from tests.test_gpu_cache8_calls import gen, ints

pytestmark = pytest.mark.gpu


def _with(v, positions, value=math.nan):
    v = v.clone()
    v[positions] = value
    return v


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 96, 256])
def test_lse_beside_value_rows_that_are_nan(gpu, code, dt, D):
    g = gen(D)
    lengths = [200, 170, 90]
    kc, vc, ks, vs, pages, seqs = paged8(g, lengths, 16, 2, D, dt, CODES[code])
    at = {0: [90, 150], 1: [168], 2: []}
    for b, rows in at.items():
        for p in rows:
            vs[pages[b, p // 16].long(), :, p % 16] = math.nan
    seqs = [(k, _with(v, at[b])) for b, (k, v) in enumerate(seqs)]
    scales = dict(k_scale=ks, v_scale=vs)
    n = [130, 7, 20]
    starts = [0, 130, 137, 157]
    q = torch.randn((157, 4, D), generator=g, device="cuda").to(dt)
    lse = torch.empty((157, 4), device="cuda")
    out = gpu.attend_prompt_paged(q, kc, vc, pages, ints(lengths), ints(starts), lse=lse, **scales)
    for b, (k, v) in enumerate(seqs):
        s = slice(starts[b], starts[b + 1])
        assert_attention(out[s], lse[s], q[s], k, v, visible(n[b], lengths[b], True, "cuda"), D ** -0.5)
    for length in (lengths, [90, 168, 90], [91, 169, 1]):
        out = gpu.attend_decode(q[:3], kc, vc, pages, ints(length), lse=lse[:3], **scales)
        for b, (k, v) in enumerate(seqs):
            m = length[b]
            assert_attention(out[b:b + 1], lse[b:b + 1], q[b:b + 1], k[:m], v[:m], visible(1, m, True, "cuda"), D ** -0.5)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,P", [(3, 64), (70, 2048)])
def test_shared_lse_beside_value_rows_that_are_nan(gpu, code, dt, B, P):
    """A NaN in the prefix and one behind it, by the decode that looks pages up and by the launches of their own."""
    g, H, D = gen(B), 2, 128
    lengths = [P + 40 if b % 2 else P // 2 for b in range(B)]
    kc, vc, ks, vs, pages, seqs = paged8(g, lengths, 16, H, D, dt, CODES[code], shared=P // 16)
    inside, behind = P // 2 + 3, P + 5
    vs[pages[0, inside // 16].long(), 1, inside % 16] = math.nan
    vs[pages[1, behind // 16].long(), 0, behind % 16] = math.nan
    q = torch.randn((B, 4, D), generator=g, device="cuda").to(dt)
    lse = torch.empty((B, 4), device="cuda")
    alone = gpu.attend_decode_workspace_size(B, 4, H, D, pages.shape[1], 16, codes=True)
    assert (gpu.attend_decode_shared_workspace_size(B, 4, H, D, pages.shape[1], 16, P // 16, codes=True) > alone) == (B == 70)
    out = gpu.attend_decode_shared(q, kc, vc, pages[0, :P // 16].clone(), pages, ints(lengths), lse=lse, k_scale=ks, v_scale=vs)
    for b in (0, 1, 2, B - 1):
        k, v = seqs[b][0], seqs[b][1].clone()
        if lengths[b] > P:
            v[inside, 1] = math.nan
            if b == 1:
                v[behind, 0] = math.nan
        assert_attention(out[b:b + 1], lse[b:b + 1], q[b:b + 1], k, v, visible(1, lengths[b], True, "cuda"), D ** -0.5)
