"""DecodeStack with attention blocks: its steps are the public calls in their order, replays equal eager
steps bit for bit, prompts leave the slots ready to decode, idle slots take no part."""

import numpy as np
import pytest

from oracle import synth
from tests._attention import assert_attention, visible
from tests._layers import to_device

pytestmark = pytest.mark.gpu

D_MODEL, HQ, HKV, D, PAGE, PAGES = 256, 4, 2, 64, 16, 40


@pytest.fixture(scope="module")
def parts(gpu):
    import torch

    gen = torch.Generator(device="cuda").manual_seed(0)
    # Rank 256: the tile layout, whose paths sum in a fixed order.
    layers = [to_device(synth.make_layer(seed=s, n_expert=8, d=D_MODEL, ff=256, max_rank=256)) for s in (1, 2)]
    assert all(L.layout == "tiles" for L in layers)
    routers = [gpu.Router(torch.randn((D_MODEL, 8), generator=gen, device="cuda"), 2) for _ in layers]
    ws = [((torch.randn((D_MODEL, (HQ + 2 * HKV) * D), generator=gen, device="cuda") / 16).bfloat16(),
           (torch.randn((HQ * D, D_MODEL), generator=gen, device="cuda") / 16).bfloat16()) for _ in layers]
    return layers, routers, ws, gpu.rope_table(200, D)


def _stack(gpu, parts, T, max_pages=8):
    import torch

    layers, routers, ws, rope = parts
    blocks = [gpu.Attention(a, b, HQ, HKV, PAGES, PAGE, rope=rope) for a, b in ws]
    s = gpu.DecodeStack(layers, routers, T, attention=blocks, max_pages=max_pages)
    order = np.random.default_rng(3).permutation(PAGES).astype(np.int32)
    s.pages.copy_(torch.from_numpy(order[:T * max_pages].reshape(T, max_pages)).cuda())
    return s


def _x(gen, n):
    import torch

    return torch.randn((n, D_MODEL), generator=gen, device="cuda")


def _ints(v):
    import torch

    return torch.tensor(v, dtype=torch.int32, device="cuda")


def test_step_is_the_public_calls_in_order(gpu, parts):
    import torch

    gen = torch.Generator(device="cuda").manual_seed(1)
    layers, routers, ws, rope = parts
    s = _stack(gpu, parts, 3)
    s.positions.copy_(_ints([0, 0, -1]))
    caches = [tuple(torch.zeros_like(a.k_cache) for _ in range(2)) for a in s.attention]
    pos = _ints([0, 0, -1])
    for _ in range(4):
        x0 = _x(gen, 3)
        got = s.forward(x0).clone()
        x = x0
        for L, r, (wqkv, wo), (kc, vc) in zip(layers, routers, ws, caches):
            qkv = (x.bfloat16() @ wqkv).view(3, HQ + 2 * HKV, D)
            q = gpu.kv_append(qkv[:, HQ:HQ + HKV], qkv[:, HQ + HKV:], kc, vc, s.pages, pos, q=qkv[:, :HQ], rope=rope)
            a = gpu.attend_decode(q, kc, vc, s.pages, pos + 1)
            assert bool((a[2] == 0).all())  # the idle slot
            for b in range(2):
                n = int(pos[b]) + 1
                at = torch.arange(n, device="cuda")
                rows = s.pages[b].long()[at // PAGE]
                assert_attention(a[b:b + 1], None, q[b:b + 1], kc[rows, at % PAGE], vc[rows, at % PAGE],
                                 visible(1, n, True, "cuda"), D ** -0.5)
            h = x + a.view(3, -1) @ wo
            ids, w = r(h)
            x = h + gpu.moe_forward(h, ids, w, L)
        assert torch.equal(got, x)
        pos = pos + (pos >= 0)
        assert torch.equal(s.positions, pos)
    for a, (kc, vc) in zip(s.attention, caches):
        assert torch.equal(a.k_cache, kc) and torch.equal(a.v_cache, vc)


def test_captured_steps_equal_eager_steps(gpu, parts):
    import torch

    gen = torch.Generator(device="cuda").manual_seed(2)
    eager, graph = _stack(gpu, parts, 4), _stack(gpu, parts, 4)
    n = [37, 5, 20]
    x = _x(gen, sum(n))
    starts, slots = _ints([0, 37, 42, 62]), _ints([2, 0, 1])  # slot 3 stays idle
    want = eager.prompt(x, starts, slots)
    assert torch.equal(graph.prompt(x, starts, slots), want)
    assert eager.positions.tolist() == [5, 20, 37, -1]
    graph.capture()
    assert graph.positions.tolist() == [5, 20, 37, -1]
    for i in range(5):
        x0 = _x(gen, 4)
        graph.load(x0)
        got = graph.replay()
        assert torch.equal(got, eager.forward(x0)), i
        torch.cuda.synchronize()
    assert graph.positions.tolist() == eager.positions.tolist() == [10, 25, 42, -1]


def test_prompt_in_chunks_attends_to_what_is_cached(gpu, parts):
    """The first layer of a chunked prompt: its cache equals the one of the whole prompt (row by row, as far as the
    projections of different batches agree), and its queries see the cached part."""
    import torch

    gen = torch.Generator(device="cuda").manual_seed(3)
    whole, chunks = _stack(gpu, parts, 2), _stack(gpu, parts, 2)
    x = _x(gen, 100)
    whole.prompt(x, _ints([0, 60, 100]), _ints([0, 1]))
    chunks.prompt(torch.cat((x[:33], x[60:75])), _ints([0, 33, 48]), _ints([0, 1]))
    chunks.prompt(torch.cat((x[75:100], x[33:60])), _ints([0, 25, 52]), _ints([1, 0]))
    assert whole.positions.tolist() == chunks.positions.tolist() == [60, 40]
    a, b = whole.attention[0], chunks.attention[0]
    for got, want in ((b.k_cache, a.k_cache), (b.v_cache, a.v_cache)):
        # Sums of 256 products in another order, rounded once: 256 * 2^-24 of their size, and a step of bf16.
        assert float((got.float() - want.float()).abs().max()) <= 2.0 ** -7 * float(want.float().abs().max())
        assert torch.equal(got == 0, want == 0)


def test_padded_prompt(gpu, parts):
    """Rows in front of the first and behind the last sequence reach no cache; the sequences' own rows are those of the call without."""
    import torch

    gen = torch.Generator(device="cuda").manual_seed(4)
    a, b = _stack(gpu, parts, 3), _stack(gpu, parts, 3)
    x = _x(gen, 40)
    for s in (a, b):  # what the padding must not touch
        s.prompt(_x(torch.Generator(device="cuda").manual_seed(5), 30), _ints([0, 20, 30]), _ints([0, 2]))
    want = a.prompt(x, _ints([4, 20, 20, 33]), _ints([0, 1, 2]))
    first = a.positions.clone()
    got = b.prompt(x[4:33], _ints([0, 16, 16, 29]), _ints([0, 1, 2]))
    assert a.positions.tolist() == [36, 0, 23] == b.positions.tolist() and torch.equal(first, a.positions)
    assert bool(torch.isfinite(want).all())
    for p, q in zip(a.attention, b.attention):
        assert torch.equal(p.k_cache == 0, q.k_cache == 0) and torch.equal(p.v_cache == 0, q.v_cache == 0)
    # The first layer's keys are the same, but for the projections' sums in another order.
    k, l = a.attention[0].k_cache.float(), b.attention[0].k_cache.float()
    assert float((k - l).abs().max()) <= 2.0 ** -7 * float(l.abs().max())
    assert want.shape == x.shape and got.shape == (29, D_MODEL)


def test_refusals(gpu, parts):
    import torch

    layers, routers, ws, rope = parts
    block = gpu.Attention(*ws[0], HQ, HKV, PAGES, PAGE, rope=rope)
    with pytest.raises(ValueError):
        gpu.DecodeStack(layers, routers, 2, attention=[block], max_pages=4)
    with pytest.raises(ValueError):
        gpu.DecodeStack(layers, routers, 2, attention=[block, block])
    with pytest.raises(ValueError):
        gpu.DecodeStack(layers, routers, 2, max_pages=4)
    with pytest.raises(RuntimeError):
        gpu.DecodeStack(layers, routers, 2).prompt(torch.zeros((1, D_MODEL), device="cuda"), _ints([0, 1]), _ints([0]))
    with pytest.raises(ValueError):
        gpu.Attention(ws[0][0], ws[0][1], 3, 2, PAGES, PAGE)
    with pytest.raises(ValueError):
        gpu.Attention(torch.zeros((64, 3 * 20), dtype=torch.bfloat16, device="cuda"),
                      torch.zeros((20, 64), dtype=torch.bfloat16, device="cuda"), 1, 1, PAGES, PAGE)  # heads of 20
    with pytest.raises(TypeError):
        gpu.Attention(ws[0][0].float(), ws[0][1].float(), HQ, HKV, PAGES, PAGE)
    s = _stack(gpu, parts, 2)
    with pytest.raises(ValueError):
        s.prompt(torch.zeros((2, D_MODEL), device="cuda"), _ints([0, 2]), _ints([0, 1]))
    for change in (0, 1, 2):
        args = [torch.zeros((2, D_MODEL), device="cuda"), _ints([0, 1, 2]), _ints([0, 1])]
        args[change] = args[change].cpu()
        with pytest.raises(ValueError, match="cuda"):
            s.prompt(*args)


def test_slots_without_room_store_nothing_more(gpu, parts):
    import torch

    gen = torch.Generator(device="cuda").manual_seed(6)
    s = _stack(gpu, parts, 2, max_pages=2)  # 32 positions a slot
    s.prompt(_x(gen, 50), _ints([0, 30, 50]), _ints([0, 1]))
    for i in range(4):
        if i == 2:
            before = [(a.k_cache.clone(), a.v_cache.clone()) for a in s.attention]
        out = s.forward(_x(gen, 2)).clone()
        assert bool(torch.isfinite(out).all())
    assert s.positions.tolist() == [34, 24]
    mine = s.pages[0].long()
    for a, (k, v) in zip(s.attention, before):
        assert torch.equal(a.k_cache[mine], k[mine]) and torch.equal(a.v_cache[mine], v[mine])
        assert not torch.equal(a.k_cache[s.pages[1].long()], k[s.pages[1].long()])


def test_slots_behind_their_rotation_table_read_what_is_stored(gpu, parts):
    """A table that ends (at 20) before the pages do (at 32): its slot's later tokens are not stored, and the rows behind it, here
    NaN, reach nothing: those tokens' attention is zeros, the other slot's its own.  Eager and captured."""
    import torch

    layers, routers, ws, _ = parts
    short = (layers, routers, ws, gpu.rope_table(20, D))
    gen = torch.Generator(device="cuda").manual_seed(7)
    x, steps = _x(gen, 23), [_x(gen, 2) for _ in range(5)]
    for captured in (False, True):
        s = _stack(gpu, short, 2, max_pages=2)
        for a in s.attention:
            a.k_cache.fill_(float("nan")), a.v_cache.fill_(float("nan"))
        s.prompt(x, _ints([0, 18, 23]), _ints([0, 1]))
        if captured:
            s.capture()
        for i, x0 in enumerate(steps):
            s.load(x0)
            out = s.replay() if captured else s.forward()
            torch.cuda.synchronize()
            assert bool(torch.isfinite(out).all()), i
            a = s.attention[0]
            qkv = (x0.bfloat16() @ a.w_qkv).view(2, HQ + 2 * HKV, D)
            q = gpu.kv_append(qkv[:, HQ:HQ + HKV], qkv[:, HQ + HKV:], a.k_cache.clone(), a.v_cache.clone(), s.pages, _ints([18 + i, 5 + i]),
                              q=qkv[:, :HQ], rope=a.rope, q_out=qkv[:, :HQ])
            y = gpu.attend_decode(q, a.k_cache, a.v_cache, s.pages, _ints([19 + i if i < 2 else 0, 6 + i]))
            assert torch.equal(s.h[0], x0 + y.view(2, -1) @ a.w_o), i
            assert i < 2 or torch.equal(s.h[0][0], x0[0])
        assert s.positions.tolist() == [23, 10]
        for a in s.attention:
            for t in (a.k_cache, a.v_cache):
                rows = t[s.pages[0].long()].view(32, HKV, D)
                assert bool(torch.isfinite(rows[:20]).all()) and bool(torch.isnan(rows[20:]).all())
        # A prompt that passes the table reads no such row either.
        assert bool(torch.isfinite(s.prompt(x, _ints([0, 2, 23]), _ints([0, 1]))).all())


def test_prompts_that_pass_the_rotation_table(gpu, parts):
    """Tokens in the table see what they would in a longer one; those behind it get zeros; other sequences are their own."""
    import torch

    gen = torch.Generator(device="cuda").manual_seed(10)
    w_qkv, eye = parts[2][0][0], torch.eye(D_MODEL, dtype=torch.bfloat16, device="cuda")  # w_o: the attention as it is
    order = torch.randperm(PAGES, generator=gen, device="cuda").int()
    pages = torch.stack((order[:4], order[4:8]))
    blocks = [gpu.Attention(w_qkv, eye, HQ, HKV, PAGES, PAGE, rope=gpu.rope_table(n, D)) for n in (41, 64)]
    for a in blocks:
        a.k_cache.fill_(float("nan")), a.v_cache.fill_(float("nan"))
    first = [0, 0]
    for new in ([30, 12], [25, 7]):  # positions 30 .. 54 and 12 .. 18: the first passes 41
        T, starts = sum(new), _ints([0, new[0], sum(new)])
        x = _x(gen, T)
        pos = _ints([f + i for f, n in zip(first, new) for i in range(n)])
        seqs, lengths = _ints([0] * new[0] + [1] * new[1]), _ints([f + n for f, n in zip(first, new)])
        got, whole = (a.prompt(x, pages, pos, seqs, starts, lengths).view(T, HQ, D) for a in blocks)
        b = blocks[1]
        q = (x.bfloat16() @ w_qkv).view(T, HQ + 2 * HKV, D)[:, :HQ]
        q = gpu.kv_append(q[:, :HKV], q[:, :HKV], b.k_cache.clone(), b.v_cache.clone(), pages, pos, seqs=seqs, q=q, rope=b.rope)
        for i, (f, n) in enumerate(zip(first, new)):
            at = torch.arange(f + n, device="cuda")
            p, o = pages[i].long()[at // PAGE], at % PAGE
            r, seen = int(starts[i]), min(n, 41 - f)
            for y, m in ((got, seen), (whole, n)):
                assert_attention(y[r:r + m], None, q[r:r + m], b.k_cache[p, o], b.v_cache[p, o], visible(n, f + n, True, "cuda")[:m], D ** -0.5)
            assert bool((got[r + seen:r + n] == 0).all())
        first = [f + n for f, n in zip(first, new)]
    rows = blocks[0].k_cache[pages[0].long()].view(64, HKV, D)
    assert bool(torch.isfinite(rows[:41]).all()) and bool(torch.isnan(rows[41:]).all())


def test_blocks_that_share_a_cache_are_refused(gpu, parts):
    """Layers that store into one cache would read each other's keys."""
    layers, routers, ws, rope = parts
    make = lambda i: gpu.Attention(*ws[i], HQ, HKV, PAGES, PAGE, rope=rope)
    block = make(0)
    with pytest.raises(ValueError, match="cache of its own"):
        gpu.DecodeStack(layers, routers, 2, attention=[block, block], max_pages=4)
    for name in ("k_cache", "v_cache"):
        other = make(1)
        setattr(other, name, getattr(block, name).view(PAGES, PAGE, HKV, D))
        with pytest.raises(ValueError, match="cache of its own"):
            gpu.DecodeStack(layers, routers, 2, attention=[block, other], max_pages=4)
    other = make(1)
    other.v_cache = other.k_cache
    with pytest.raises(ValueError, match="cache of its own"):
        gpu.DecodeStack(layers, routers, 2, attention=[block, other], max_pages=4)
    gpu.DecodeStack(layers, routers, 2, attention=[make(0), make(0)], max_pages=4)  # shared weights are no matter


def test_prompts_without_slots_or_tokens(gpu, parts):
    """Rows of no sequence pass the experts alone, also where there is no sequence at all; a sequence of no tokens starts an idle
    slot at 0, whether or not other rows come with it."""
    import torch

    gen = torch.Generator(device="cuda").manual_seed(8)
    layers, routers, _, _ = parts
    s = _stack(gpu, parts, 3)
    s.prompt(_x(gen, 9), _ints([0, 9]), _ints([2]))
    before = [(a.k_cache.clone(), a.v_cache.clone()) for a in s.attention]
    x = _x(gen, 7)
    got = s.prompt(x, _ints([0]), _ints([]))
    want = x
    for L, r in zip(layers, routers):
        ids, w = gpu.route(r.k, x=want, router=r.weight)
        want = want + gpu.moe_forward(want, ids, w, L)
    assert torch.equal(got, want)
    assert s.positions.tolist() == [-1, -1, 9]
    assert s.prompt(x[:0], _ints([0, 0, 0]), _ints([2, 0])).shape == (0, D_MODEL)
    assert s.positions.tolist() == [0, -1, 9]
    assert torch.equal(s.prompt(x, _ints([7, 7]), _ints([1])), want)
    assert s.positions.tolist() == [0, 0, 9]
    assert s.prompt(x[:0], _ints([0]), _ints([])).shape == (0, D_MODEL)
    for a, (k, v) in zip(s.attention, before):
        assert torch.equal(a.k_cache, k) and torch.equal(a.v_cache, v)


def test_prompt_is_the_public_calls_in_order(gpu, parts):
    """A padded batch behind cached tokens, one sequence without any: rows, caches and attention of every layer, rebuilt from the
    public calls, the attention against 64 bits."""
    import torch

    gen = torch.Generator(device="cuda").manual_seed(9)
    layers, routers, ws, rope = parts
    s = _stack(gpu, parts, 4)
    s.prompt(_x(gen, 33), _ints([0, 20, 33]), _ints([3, 1]))
    caches = [(a.k_cache.clone(), a.v_cache.clone()) for a in s.attention]
    new, first, slots, lead, tail = [17, 0, 40, 1], [0, 13, 20, 0], [0, 1, 3, 2], 2, 3
    starts = [lead]
    for n in new:
        starts.append(starts[-1] + n)
    N = starts[-1] + tail
    x = x0 = _x(gen, N)
    got = s.prompt(x0, _ints(starts), _ints(slots))
    rows = [b for b, n in enumerate(new) for _ in range(n)]
    seqs = _ints([0] * lead + rows + [0] * tail)
    pos = _ints([-1] * lead + [first[b] + i for b, n in enumerate(new) for i in range(n)] + [-1] * tail)
    pages, lengths = s.pages[_ints(slots).long()], _ints([a + n for a, n in zip(first, new)])
    for L, r, (wqkv, wo), (kc, vc), a in zip(layers, routers, ws, caches, s.attention):
        qkv = (x.bfloat16() @ wqkv).view(N, HQ + 2 * HKV, D)
        q = gpu.kv_append(qkv[:, HQ:HQ + HKV], qkv[:, HQ + HKV:], kc, vc, pages, pos, seqs=seqs, q=qkv[:, :HQ], rope=rope, q_out=qkv[:, :HQ])
        y = gpu.attend_prompt_paged(q, kc, vc, pages, lengths, _ints(starts), out=torch.zeros((N, HQ, D), dtype=q.dtype, device="cuda"))
        assert bool((y[:lead] == 0).all()) and bool((y[starts[-1]:] == 0).all())
        for b, n in enumerate(new):
            at = torch.arange(first[b] + n, device="cuda")
            p, o = pages[b].long()[at // PAGE], at % PAGE
            assert_attention(y[starts[b]:starts[b + 1]], None, q[starts[b]:starts[b + 1]], kc[p, o], vc[p, o],
                             visible(n, first[b] + n, True, "cuda"), D ** -0.5)
        h = x + y.view(N, -1) @ wo
        ids, w = gpu.route(r.k, x=h, router=r.weight)
        x = h + gpu.moe_forward(h, ids, w, L)
        assert torch.equal(a.k_cache, kc) and torch.equal(a.v_cache, vc)
    assert torch.equal(got, x)
    assert s.positions[_ints(slots).long()].tolist() == lengths.tolist()


def test_blocks_without_sequences_or_tokens(gpu, parts):
    import torch

    _, _, ws, rope = parts
    a = gpu.Attention(*ws[0], HQ, HKV, PAGES, PAGE, rope=rope)
    x, pages, none = torch.empty((0, D_MODEL), device="cuda"), torch.zeros((2, 3), dtype=torch.int32, device="cuda"), _ints([])
    assert a.decode(x, pages[:0], none, none).shape == (0, D_MODEL)
    assert a.prompt(x, pages, none, none, _ints([0, 0, 0]), _ints([0, 5])).shape == (0, D_MODEL)
    assert a.prompt(x, pages[:0], none, none, _ints([0]), none).shape == (0, D_MODEL)
    y = a.prompt(torch.ones((2, D_MODEL), device="cuda"), pages[:0], _ints([-1, -1]), _ints([0, 0]), _ints([0]), none)  # padding alone
    assert y.shape == (2, D_MODEL) and bool((y == 0).all())
    assert bool((a.k_cache == 0).all()) and bool((a.v_cache == 0).all())


def test_prompts_between_replays_and_steps_on_another_stream(gpu, parts):
    """A slot is filled, retired and filled anew between the replays of one graph; an eager stack on another stream agrees."""
    import torch

    gen = torch.Generator(device="cuda").manual_seed(11)
    eager, graph = _stack(gpu, parts, 3), _stack(gpu, parts, 3)
    graph.capture()
    side = torch.cuda.Stream()

    def both(f):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            a = f(eager, eager.forward)
        torch.cuda.current_stream().wait_stream(side)

        def replay(x0):
            graph.load(x0)
            return graph.replay()

        return a, f(graph, replay)

    for starts, slots, n in (([0, 30], [1], 30), ([0, 5, 26], [2, 1], 26), ([0, 1], [0], 1), ([0, 40], [1], 40)):
        if slots == [1] and n == 40:  # retired: its pages are another sequence's
            eager.positions[1] = graph.positions[1] = -1
        x, st, sl = _x(gen, n), _ints(starts), _ints(slots)
        a, b = both(lambda s, step: s.prompt(x, st, sl))
        assert torch.equal(a, b)
        for _ in range(3):
            x0 = _x(gen, 3)
            a, b = both(lambda s, step: step(x0).clone())
            assert torch.equal(a, b) and eager.positions.tolist() == graph.positions.tolist()
    assert eager.positions.tolist() == [7, 43, 14]
    for p, q in zip(eager.attention, graph.attention):
        assert torch.equal(p.k_cache, q.k_cache) and torch.equal(p.v_cache, q.v_cache)
