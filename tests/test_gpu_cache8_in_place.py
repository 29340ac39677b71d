"""Queries rotated where they stand, beside keys and values on their way into an 8-bit cache: the same bits as into another tensor."""

import pytest
import torch

from tests._cache8 import CODES, bits, empty_cache
from tests.test_gpu_cache8_calls import gen, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("T,Hq", [(1, 4), (300, 8), (900, 16)])
@pytest.mark.parametrize("D,rot,interleaved", [(128, 128, False), (64, 64, True), (128, 20, False), (112, 102, True), (256, 250, False), (48, 12, True), (80, 72, False), (16, 2, False)])
def test_queries_rotated_in_place(gpu, code, D, rot, interleaved, T, Hq):
    g = gen(D + T)
    q, k, v = (torch.randn((T, h, D), generator=g, device="cuda").half() for h in (Hq, 2, 2))
    table = gpu.rope_table(T + 3, rot)
    pages = torch.arange(-(-(T + 3) // 8), dtype=torch.int32, device="cuda")[None]
    at, seqs = torch.arange(3, T + 3, dtype=torch.int32, device="cuda"), ints([0] * T)
    got = []
    for in_place in (False, True):
        (kc, ks), (vc, vs) = (empty_cache(pages.shape[1], 8, 2, D, CODES[code]) for _ in range(2))
        mine = q.clone()
        out = gpu.kv_append(k, v, kc, vc, pages, at, seqs=seqs, q=mine, rope=table, interleaved=interleaved, q_out=mine if in_place else None, k_scale=ks, v_scale=vs)
        assert (out is mine) == in_place and (in_place or torch.equal(mine, q))
        got.append((out, bits(kc), bits(vc), ks.nan_to_num(-1.0), vs.nan_to_num(-1.0)))
    assert all(torch.equal(a, b) for a, b in zip(*got))
