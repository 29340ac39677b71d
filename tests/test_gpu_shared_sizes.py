"""attend_decode_shared over 16-bit caches whose pages and heads no 8-bit one has."""

import pytest
import torch

from tests._attention import assert_attention, paged

pytestmark = pytest.mark.gpu
DT = {"f16": torch.float16, "bf16": torch.bfloat16}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("shared,lengths,Hkv,G,D,page,order", [
    (3, [20, 15, 0, 7, 33], 2, 3, 8, 5, "rows"), (40, [41, 40, 100, 1], 1, 4, 24, 1, "heads"), (7, [100, 91, 92, 60], 3, 1, 72, 13, "rows"),
    (2, [300, 25, 24], 1, 2, 200, 12, "heads"), (100, [1301, 1299, 1300, 700], 1, 17, 248, 13, "rows"),
    # The prefix by itself.
    (200, [2600 + i for i in range(70)], 2, 2, 136, 13, "rows"), (1700, [1700, 1712, 1699, 3, 0] * 30, 2, 3, 72, 1, "rows"), (150, [1801, 1950] * 150, 1, 9, 24, 12, "heads")])
def test_pages_and_heads_of_16_bit_caches(gpu, dt, shared, lengths, Hkv, G, D, page, order):
    g, dt, n = gen(D + page), DT[dt], shared * page
    kc, vc, own, seqs = paged(g, [n] + [max(0, m - n) for m in lengths], page, Hkv, D, dt, order=order)
    prefix = own[0, :shared].contiguous()
    pages = torch.cat((torch.full((len(lengths), shared), -3, dtype=torch.int32, device="cuda"), own[1:]), 1)
    B, H = len(lengths), Hkv * G
    q = torch.randn((B, H, D), generator=g, device="cuda").to(dt)
    lse = torch.empty((B, H), device="cuda")
    out = gpu.attend_decode_shared(q, kc, vc, prefix, pages, ints(lengths), lse=lse)
    for b in {*range(min(B, 12)), B - 1}:
        k, v = (torch.cat((c, o))[:lengths[b]] for c, o in zip(seqs[0], seqs[1 + b]))
        assert_attention(out[b:b + 1], lse[b:b + 1], q[b:b + 1], k, v, torch.ones((1, lengths[b]), dtype=torch.bool, device="cuda"), D ** -0.5)
