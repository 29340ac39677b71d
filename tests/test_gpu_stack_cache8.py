"""DecodeStack with 8-bit caches, shared prefixes and norms: its steps are the public calls in their order, replays equal eager
steps bit for bit, a step over a shared prefix is the step over pages of one's own to rounding."""

import numpy as np
import pytest
import torch

from oracle import synth
from tests._attention import assert_attention, visible
from tests._cache8 import values
from tests._layers import to_device

pytestmark = pytest.mark.gpu

D_MODEL, HQ, HKV, D, PAGE, PAGES = 256, 4, 2, 64, 16, 60
CACHES = {"16": None, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}


@pytest.fixture(scope="module")
def parts(gpu):
    gen = torch.Generator(device="cuda").manual_seed(0)
    # Rank 256: the tile layout, whose paths sum in a fixed order.
    layers = [to_device(synth.make_layer(seed=s, n_expert=8, d=D_MODEL, ff=256, max_rank=256)) for s in (1, 2)]
    routers = [gpu.Router(torch.randn((D_MODEL, 8), generator=gen, device="cuda"), 2) for _ in layers]
    ws = [((torch.randn((D_MODEL, (HQ + 2 * HKV) * D), generator=gen, device="cuda") / 16).bfloat16(),
           (torch.randn((HQ * D, D_MODEL), generator=gen, device="cuda") / 16).bfloat16()) for _ in layers]
    r = lambda: torch.randn(D_MODEL, generator=gen, device="cuda")  # noqa: E731
    norms = [gpu.BlockNorm(pre=gpu.Norm(1 + 0.1 * r()), post=gpu.Norm(1 + 0.1 * r()), gate=0.5 * r()),
             gpu.BlockNorm(pre=gpu.Norm(1 + 0.1 * r(), bias=0.1 * r(), kind="layer"), scale=0.7),
             gpu.BlockNorm(post=gpu.Norm(), scale=0.5), gpu.BlockNorm(pre=gpu.Norm((1 + 0.1 * r()).bfloat16()), gate=r().bfloat16())]
    return layers, routers, ws, norms


def _stack(gpu, parts, T, cache="int8", norms=True, max_pages=8, seed=3):
    layers, routers, ws, ns = parts
    blocks = [gpu.Attention(a, b, HQ, HKV, PAGES, PAGE, rope=gpu.rope_table(max_pages * PAGE, D), cache_dtype=CACHES[cache]) for a, b in ws]
    s = gpu.DecodeStack(layers, routers, T, attention=blocks, max_pages=max_pages, norms=ns if norms else None)
    order = np.random.default_rng(seed).permutation(PAGES).astype(np.int32)
    s.pages.copy_(torch.from_numpy(order[:T * max_pages].reshape(T, max_pages)).cuda())
    return s


def _x(gen, n):
    return torch.randn((n, D_MODEL), generator=gen, device="cuda")


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("norms", [True, False])
def test_step_is_the_public_calls_in_order(gpu, parts, cache, norms):
    gen = torch.Generator(device="cuda").manual_seed(1)
    layers, routers, ws, ns = parts
    s, own = _stack(gpu, parts, 3, cache, norms), _stack(gpu, parts, 3, cache, norms)
    pos = _ints([0, 0, -1])
    s.positions.copy_(pos)
    for _ in range(4):
        x = x0 = _x(gen, 3)
        got = s.forward(x0).clone()
        n = gpu.residual_norm(x, pre=ns[0].pre, dtype=torch.bfloat16)[1] if norms else x
        for l, (L, r, (wqkv, wo), a) in enumerate(zip(layers, routers, ws, own.attention)):
            qkv = (n.bfloat16() @ wqkv).view(3, HQ + 2 * HKV, D)
            scales = dict(k_scale=a.k_scale, v_scale=a.v_scale)
            q = gpu.kv_append(qkv[:, HQ:HQ + HKV], qkv[:, HQ + HKV:], a.k_cache, a.v_cache, s.pages, pos, q=qkv[:, :HQ], rope=a.rope, **scales)
            y = gpu.attend_decode(q, a.k_cache, a.v_cache, s.pages, pos + 1, **scales)
            assert bool((y[2] == 0).all())  # the idle slot
            for b in range(2):
                m = int(pos[b]) + 1
                at, seq = torch.arange(m, dtype=torch.int32, device="cuda"), torch.full((m,), b, dtype=torch.int32, device="cuda")
                if cache == "16":
                    k, v = gpu.kv_read(a.k_cache, a.v_cache, s.pages, at, seqs=seq)
                else:  # unrounded
                    rows = s.pages[b].long()[at.long() // PAGE]
                    k, v = (values(c.float()[rows, at.long() % PAGE], z[rows, :, at.long() % PAGE])
                            for c, z in ((a.k_cache, a.k_scale), (a.v_cache, a.v_scale)))
                assert_attention(y[b:b + 1], None, q[b:b + 1], k, v, visible(1, m, True, "cuda"), D ** -0.5)
            y = y.view(3, -1) @ wo
            if norms:
                i = 2 * l
                x, n = gpu.residual_norm(x, y, post=ns[i].post, gate=ns[i].gate, scale=ns[i].scale, pre=ns[i + 1].pre, dtype=torch.float32)
            else:
                x = n = x + y
            ids, w = r(n)
            y = gpu.moe_forward(n, ids, w, L)
            if norms:
                i += 1
                x, n = gpu.residual_norm(x, y, post=ns[i].post, gate=ns[i].gate, scale=ns[i].scale, pre=ns[i + 1].pre if i < 3 else None, dtype=torch.bfloat16)
                n = x if n is None else n
            else:
                x = n = x + y
        assert torch.equal(got, x)
        pos = pos + (pos >= 0)
        assert torch.equal(s.positions, pos)
    for a, b in zip(s.attention, own.attention):
        assert torch.equal(a.k_cache.view(torch.uint8), b.k_cache.view(torch.uint8)) and torch.equal(a.v_cache.view(torch.uint8), b.v_cache.view(torch.uint8))


@pytest.mark.parametrize("cache", CACHES)
def test_captured_steps_equal_eager_steps_over_a_shared_prefix(gpu, parts, cache):
    gen = torch.Generator(device="cuda").manual_seed(2)
    eager, graph, plain = (_stack(gpu, parts, 4, cache) for _ in range(3))
    prefix = _ints([59, 3, 41])
    n = [3 * PAGE, 5, 20]
    x = _x(gen, sum(n))
    for s in (eager, graph, plain):
        if s is plain:
            s.pages[:, :3] = prefix
        else:
            s.share(prefix)
            assert bool((s.pages[:, :3] == prefix).all())
        s.prompt(x[:48], _ints([0, 48]), _ints([2]))  # the prefix, through one slot
        s.positions.copy_(_ints([48, 48, 48, -1]))
        s.prompt(x[48:], _ints([0, 5, 25]), _ints([1, 0]))
    assert eager.positions.tolist() == [68, 53, 48, -1]
    graph.capture()
    for i in range(5):
        x0 = _x(gen, 4)
        graph.load(x0)
        got = graph.replay()
        assert torch.equal(got, eager.forward(x0)), i
        if i == 0:  # one layer's attention was summed otherwise; a router may turn on a rounding later on
            want = plain.forward(x0)
            assert float((got[:3] - want[:3]).norm() / want[:3].norm()) < 0.05
        torch.cuda.synchronize()
        graph.positions.mul_(1)  # the program's own work between replays
    assert graph.positions.tolist() == eager.positions.tolist() == [73, 58, 53, -1]
    graph.share(None)
    assert graph.graph is None and graph.prefix is None
    eager.share(None)
    assert torch.equal(graph.forward(x0), eager.forward(x0))


def test_shared_steps_are_steps_over_the_same_pages(gpu, parts):
    """One layer's attention, shared and not, of the same cache: each within the tolerance of the 64-bit one, so within their sum."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    a = _stack(gpu, parts, 4, "int8").attention[0]
    pages = torch.cat((_ints([[7, 8]] * 4), _ints(range(10, 26)).view(4, 4)), 1)
    for b in range(4):
        n = 32 + 11 * b if b else 60
        a.prompt(_x(gen, n), pages, _ints(range(n)), _ints([b] * n), _ints([0] * (b + 1) + [n] * (4 - b)), _ints([n if i == b else 0 for i in range(4)]))
    lengths = _ints([60, 43, 20, 0])
    q = torch.randn((4, HQ, D), generator=gen, device="cuda").bfloat16()
    scales = dict(k_scale=a.k_scale, v_scale=a.v_scale)
    out = gpu.attend_decode_shared(q, a.k_cache, a.v_cache, _ints([7, 8]), pages, lengths, **scales)
    for b in range(4):
        m = int(lengths[b])
        at = torch.arange(m, device="cuda")
        rows = pages[b].long()[at // PAGE]
        k, v = (values(c.float()[rows, at % PAGE], z[rows, :, at % PAGE]) for c, z in ((a.k_cache, a.k_scale), (a.v_cache, a.v_scale)))
        for got in (out, gpu.attend_decode(q, a.k_cache, a.v_cache, pages, lengths, **scales)):
            assert_attention(got[b:b + 1], None, q[b:b + 1], k, v, visible(1, m, False, "cuda"), D ** -0.5)


def test_prompts_with_norms(gpu, parts):
    """A prompt's last token, and the same tokens one step at a time; padding, no sequences and no tokens."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    s = _stack(gpu, parts, 2)
    x = _x(gen, 9)
    out = s.prompt(x, _ints([2, 9]), _ints([1]))
    assert out.shape == (9, D_MODEL) and bool(torch.isfinite(out).all()) and s.positions.tolist() == [-1, 7]
    # Padded rows' attention is zeros: as without sequences.
    alone = s.prompt(x, _ints([0]), _ints([]))
    assert torch.equal(out[:2], alone[:2])
    assert s.prompt(x[:0], _ints([0]), _ints([])).shape == (0, D_MODEL)


def test_experts_alone_with_norms(gpu, parts):
    layers, routers, _, ns = parts
    s = gpu.DecodeStack(layers, routers, 3, norms=[ns[0], ns[3]])
    x = x0 = _x(torch.Generator(device="cuda").manual_seed(6), 3)
    n = gpu.residual_norm(x, pre=ns[0].pre, dtype=torch.float32)[1]
    for l, (b, nxt) in enumerate(((ns[0], ns[3]), (ns[3], None))):
        ids, w = routers[l](n)
        x, n = gpu.residual_norm(x, gpu.moe_forward(n, ids, w, layers[l]), post=b.post, gate=b.gate, scale=b.scale, pre=nxt.pre if nxt else None, dtype=torch.float32)
    assert torch.equal(s.forward(x0), x)
    s.capture()
    s.load(x0)
    for _ in range(3):
        assert torch.equal(s.replay(), x)
        torch.cuda.synchronize()


def test_refusals(gpu, parts):
    layers, routers, ws, ns = parts
    for kw, error in ((dict(cache_dtype=torch.float16), TypeError), (dict(cache_dtype=torch.float32), TypeError), (dict(cache_dtype=torch.int8, page_size=12), ValueError)):
        with pytest.raises(error):
            gpu.Attention(*ws[0], HQ, HKV, **{**dict(n_pages=4, page_size=16), **kw})
    w = torch.zeros((64, 3 * 40), dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError):
        gpu.Attention(w, torch.zeros((40, 64), dtype=torch.float16, device="cuda"), 1, 1, 4, 16, cache_dtype=torch.int8)
    for bad in (ns[:3], ns + ns):
        with pytest.raises(ValueError):
            gpu.DecodeStack(layers, routers, 2, attention=_stack(gpu, parts, 2).attention, max_pages=4, norms=bad)
    with pytest.raises(TypeError):
        gpu.DecodeStack(layers, routers, 2, norms=[gpu.Norm(), gpu.Norm()])
    s = _stack(gpu, parts, 2)
    for bad in (torch.zeros(2, device="cuda"), _ints([[1]]), _ints([1] * 9), torch.zeros(1, dtype=torch.int32)):
        with pytest.raises(ValueError):
            s.share(bad)
    with pytest.raises(RuntimeError):
        gpu.DecodeStack(layers, routers, 2).share(_ints([1]))
