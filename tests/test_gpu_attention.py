"""kv_append, attend_decode, attend_prompt and attend_prompt_paged against plain
attention in 64 bits (tests/_attention.py, where the tolerances are derived)."""

import math

import pytest

from tests._attention import W, assert_attention, half_step, paged, visible

pytestmark = pytest.mark.gpu

DT = {"f16": "float16", "bf16": "bfloat16"}


def _dt(name):
    import torch

    return getattr(torch, DT[name])


def _gen(seed):
    import torch

    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape, dt, by=1.0):
    import torch

    return (torch.randn(shape, generator=gen, device="cuda") * by).to(dt)


def _ints(v):
    import torch

    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ---- append -------------------------------------------------------------------
def _turn64(x, rope, pos, inter):
    """x [T, H, D] rotated in 64 bits, and the tolerance of a rounded fp32 rotation."""
    import torch

    y, tol = x.double().clone(), torch.zeros_like(x, dtype=torch.float64)
    if rope is not None:
        half = rope.shape[2]
        i = torch.arange(half, device=x.device)
        a, b = (2 * i, 2 * i + 1) if inter else (i, i + half)
        c, s = rope[pos.long(), 0].double()[:, None], rope[pos.long(), 1].double()[:, None]
        xa, xb = x.double()[..., a], x.double()[..., b]
        y[..., a], y[..., b] = xa * c - xb * s, xb * c + xa * s
        tol[..., a] = 2 * W * ((xa * c).abs() + (xb * s).abs())
        tol[..., b] = 2 * W * ((xb * c).abs() + (xa * s).abs())
        tol = tol + half_step(x.dtype) * (y.abs() + tol) + torch.finfo(x.dtype).smallest_normal * half_step(x.dtype) * (tol > 0)
    return y, tol


@pytest.mark.parametrize("T,B,Hq,Hkv,D,rot,inter,page,dtype,order", [
    (1, 1, 32, 8, 128, 128, False, 16, "bf16", "rows"),
    (5, 3, 4, 2, 64, 32, True, 1, "f16", "heads"),
    (7, 2, 3, 1, 24, 20, False, 3, "bf16", "rows"),     # one pair a thread
    (6, 2, 2, 2, 40, 6, True, 5, "f16", "heads"),
    (9, 4, 5, 5, 256, 256, True, 7, "bf16", "rows"),
    (33, 2, 0, 3, 96, 48, False, 8, "f16", "rows"),     # keys and values only
    (4, 4, 2, 1, 16, 0, False, 4, "bf16", "rows"),      # no rotation
    (700, 3, 28, 4, 128, 64, False, 48, "bf16", "rows"),  # four heads a thread, 36 head rows
    (900, 3, 21, 3, 80, 80, True, 16, "f16", "heads"),    # 27 head rows: the last thread has three
])
def test_append_stores_rotated_rows(gpu, T, B, Hq, Hkv, D, rot, inter, page, dtype, order):
    import torch

    dt, gen = _dt(dtype), _gen(T)
    far = max(2 * T // B + 2, 20)
    kc, vc, pages, _ = paged(gen, [far] * B, page, Hkv, D, dt, order=order)
    qkv = _randn(gen, T, Hq + 2 * Hkv, D, dt=dt)
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    seqs = _ints([t % B for t in range(T)])
    pos = _ints([(t // B) * 2 + t % 2 for t in range(T)])
    rope = gpu.rope_table(far, rot) if rot else None
    want_k, want_v = kc.clone(), vc.clone()
    got = gpu.kv_append(k, v, kc, vc, pages, pos, seqs=seqs, q=q if Hq else None, rope=rope, interleaved=inter)
    rows = pages[seqs.long(), pos.long() // page].long()
    k64, tol = _turn64(k, rope, pos, inter)
    stored = kc[rows, pos.long() % page]
    assert float(((stored.double() - k64).abs() - tol).max()) <= 0
    assert torch.equal(vc[rows, pos.long() % page], v)
    want_k[rows, pos.long() % page], want_v[rows, pos.long() % page] = stored, v
    assert torch.equal(kc.contiguous().view(torch.int16), want_k.contiguous().view(torch.int16))  # NaN rows elsewhere, untouched
    assert torch.equal(vc.contiguous().view(torch.int16), want_v.contiguous().view(torch.int16))
    if Hq:
        q64, tol = _turn64(q, rope, pos, inter)
        assert got.shape == q.shape and float(((got.double() - q64).abs() - tol).max()) <= 0
        again = q.clone()  # in place
        assert gpu.kv_append(k, v, kc, vc, pages, pos, seqs=seqs, q=again, rope=rope, interleaved=inter, q_out=again) is again
        assert torch.equal(again, got)
    else:
        assert got is None


@pytest.mark.parametrize("D", [32, 24])
def test_append_leaves_out_what_has_no_place(gpu, D):
    """Negative and far positions, sequences and pages that do not exist, table rows that end."""
    import torch

    gen, dt, page = _gen(1), torch.bfloat16, 4
    kc, vc, pages, _ = paged(gen, [12, 8], page, 1, D, dt, width=3)
    pages[0, 1], pages[1, 0] = -7, kc.shape[0]
    before = kc.clone(), vc.clone()
    #       stored, no page, stored, bad page, seq -1, seq 2, pos -1, beyond pages, beyond the table
    seqs = [0, 0, 0, 1, -1, 2, 0, 0, 0]
    pos = [0, 5, 11, 2, 3, 3, -1, 12, 15]
    T = len(seqs)
    k, v, q = (_randn(gen, T, 1, D, dt=dt) for _ in range(3))
    rope = gpu.rope_table(14, 8)
    out = torch.full_like(q, 7.0)
    gpu.kv_append(k, v, kc, vc, pages, _ints(pos), seqs=_ints(seqs), q=q, rope=rope, q_out=out)
    for t in (0, 2):
        at = int(pages[0, pos[t] // page]), pos[t] % page
        k64, tol = _turn64(k[t:t + 1], rope, _ints(pos[t:t + 1]), False)
        assert float(((kc[at].double() - k64[0]).abs() - tol[0]).max()) <= 0 and torch.equal(vc[at], v[t])
        kc[at], vc[at] = before[0][at], before[1][at]
    assert torch.equal(kc.view(torch.int16), before[0].view(torch.int16))
    assert torch.equal(vc.view(torch.int16), before[1].view(torch.int16))
    fine = torch.tensor([0 <= p < 14 for p in pos], device="cuda")
    assert bool((out[~fine] == 7.0).all())
    q64, tol = _turn64(q[fine], rope, _ints(pos)[fine], False)
    assert float(((out[fine].double() - q64).abs() - tol).max()) <= 0


@pytest.mark.parametrize("D", [32, 24])
def test_append_with_an_empty_table_leaves_all_out(gpu, D):
    """No position is in a table without rows: nothing is stored, q_out stays."""
    import torch

    gen, dt = _gen(35), torch.bfloat16
    kc, vc, pages, _ = paged(gen, [12], 4, 1, D, dt)
    before = kc.clone(), vc.clone()
    q, k, v = (_randn(gen, 3, 1, D, dt=dt) for _ in range(3))
    out = torch.full_like(q, 7.0)
    gpu.kv_append(k, v, kc, vc, pages, _ints([0, 1, 5]), seqs=_ints([0, 0, 0]), q=q, rope=gpu.rope_table(0, 8), q_out=out)
    assert bool((out == 7.0).all())
    for got, want in zip((kc, vc), before):
        assert torch.equal(got.view(torch.int16), want.view(torch.int16))


def test_append_without_tokens_or_sequences(gpu):
    import torch

    gen, dt = _gen(2), torch.float16
    kc, vc, pages, _ = paged(gen, [4], 4, 1, 16, dt)
    none = torch.empty((0, 1, 16), dtype=dt, device="cuda")
    assert gpu.kv_append(none, none, kc, vc, pages, _ints([])) is None
    k = _randn(gen, 1, 1, 16, dt=dt)
    before = kc.clone()
    gpu.kv_append(k, k, kc, vc, pages[:0], _ints([0]), seqs=_ints([0]))
    assert torch.equal(kc.view(torch.int16), before.view(torch.int16))


# ---- decode -------------------------------------------------------------------
def _decode_check(gpu, q, kc, vc, pages, lengths, seqs, lens, scale=None, **kw):
    import torch

    lse = torch.full(q.shape[:2], 5.0, device="cuda")
    out = gpu.attend_decode(q, kc, vc, pages, lengths, scale=scale, lse=lse, **kw)
    scale = q.shape[2] ** -0.5 if scale is None else scale
    for b, n in enumerate(lens):
        k, v = seqs[b]
        assert_attention(out[b:b + 1], lse[b:b + 1], q[b:b + 1], k[:n], v[:n], visible(1, n, True, "cuda"), scale)
    return out


@pytest.mark.parametrize("lens", [(1,), (0,), (31, 32, 33), (127, 128, 129, 0, 1), (0, 0, 700, 5, 0, 2049, 1, 0)])
@pytest.mark.parametrize("Hq,Hkv,D,page,dtype", [
    (8, 2, 128, 16, "bf16"), (5, 5, 64, 8, "f16"), (16, 1, 256, 32, "bf16"), (21, 3, 96, 24, "f16"), (20, 1, 72, 1, "bf16"),
    (3, 1, 8, 3, "f16"), (40, 1, 128, 64, "f16"), (66, 2, 200, 7, "bf16"), (34, 2, 64, 16, "bf16"), (25, 1, 256, 40, "f16"),
])
def test_decode_matches_plain_attention(gpu, lens, Hq, Hkv, D, page, dtype):
    import torch

    dt, gen = _dt(dtype), _gen(sum(lens) + D)
    kc, vc, pages, seqs = paged(gen, lens, page, Hkv, D, dt)  # unused rows hold NaN
    q = _randn(gen, len(lens), Hq, D, dt=dt, by=2.0)
    out = _decode_check(gpu, q, kc, vc, pages, _ints(lens), seqs, lens)
    assert torch.equal(out, gpu.attend_decode(q, kc, vc, pages, _ints(lens)))  # equal calls, equal bits


@pytest.mark.parametrize("B,L,Hq,Hkv,D", [(1, 40001, 8, 1, 128), (3, 9000, 4, 4, 64), (300, 150, 4, 2, 64), (1100, 40, 2, 1, 32)])
def test_decode_split_over_the_chip(gpu, B, L, Hq, Hkv, D):
    """Spans that cut sequences, many sequences in a span, more sequences than workgroups."""
    import torch

    gen = _gen(B)
    lens = [max(0, L - (b * 37) % (L + 3)) for b in range(B)]
    kc, vc, pages, seqs = paged(gen, lens, 16, Hkv, D, torch.bfloat16)
    q = _randn(gen, B, Hq, D, dt=torch.bfloat16, by=3.0)
    out = gpu.attend_decode(q, kc, vc, pages, _ints(lens))
    for b in (range(B) if B < 10 else (0, 1, B // 2, B - 2, B - 1)):
        n = lens[b]
        assert_attention(out[b:b + 1], None, q[b:b + 1], *(x[:n] for x in seqs[b]), visible(1, n, True, "cuda"), D ** -0.5)


def test_decode_masks_pages_that_do_not_exist(gpu):
    import torch

    gen, dt, page, D = _gen(4), torch.bfloat16, 16, 64
    for order in ("rows", "heads"):
        kc, vc, pages, seqs = paged(gen, [200, 64, 16], page, 2, D, dt, order=order)
        q = _randn(gen, 3, 6, D, dt=dt)
        pages[0, 3], pages[0, 7], pages[2, 0] = -1, kc.shape[0] + 5, 1 << 30
        lse = torch.empty((3, 6), device="cuda")
        out = gpu.attend_decode(q, kc, vc, pages, _ints([200, 64, 16]), lse=lse, scale=0.25)
        seen = torch.ones((1, 200), dtype=torch.bool, device="cuda")
        seen[0, 48:64] = seen[0, 112:128] = False
        assert_attention(out[:1], lse[:1], q[:1], *seqs[0], seen, 0.25)
        assert_attention(out[1:2], lse[1:2], q[1:2], *seqs[1], visible(1, 64, True, "cuda"), 0.25)
        assert bool((out[2] == 0).all()) and bool((lse[2] == -math.inf).all())


def test_decode_clamps_lengths(gpu):
    import torch

    gen, dt = _gen(5), torch.float16
    kc, vc, pages, seqs = paged(gen, [64, 64], 16, 1, 64, dt)
    q = _randn(gen, 2, 4, 64, dt=dt)
    got = gpu.attend_decode(q, kc, vc, pages, _ints([1 << 30, -5]))
    assert torch.equal(got[0], gpu.attend_decode(q, kc, vc, pages, _ints([64, 0]))[0]) and bool((got[1] == 0).all())


def test_decode_infinite_and_nan_keys_reach_their_own_rows_only(gpu):
    import torch

    gen, dt = _gen(6), torch.bfloat16
    lens = [100, 100]
    kc, vc, pages, seqs = paged(gen, lens, 16, 1, 64, dt)
    q = _randn(gen, 2, 4, 64, dt=dt)
    clean = gpu.attend_decode(q, kc, vc, pages, _ints(lens))
    kc[pages[0, 2].long(), 3, 0, 5] = math.nan
    got = gpu.attend_decode(q, kc, vc, pages, _ints(lens))
    assert torch.isnan(got[0]).all() and torch.equal(got[1], clean[1])
    # A row whose scores are all -inf has nothing to weigh: zeros.
    q0 = torch.ones((1, 4, 64), dtype=dt, device="cuda")
    kc2, vc2, pages2, _ = paged(gen, [40], 16, 1, 64, dt)
    kc2[pages2[0, :3].long()] = -math.inf
    lse = torch.empty((1, 4), device="cuda")
    assert bool((gpu.attend_decode(q0, kc2, vc2, pages2, _ints([40]), lse=lse) == 0).all()) and bool((lse == -math.inf).all())


@pytest.mark.parametrize("length", [100, 3000])
def test_decode_infinite_and_nan_values_reach_their_own_rows_only(gpu, length):
    import torch

    gen, dt, D = _gen(30), torch.float16, 128
    lens = [length, length - 1]
    kc, vc, pages, seqs = paged(gen, lens, 16, 2, D, dt)
    q = _randn(gen, 2, 6, D, dt=dt)
    for key, x in ((length - 2, math.nan), (17, math.inf), (0, -math.inf)):
        seqs[1][1][key, 1, 5] = x
        vc[pages[1, key // 16].long(), key % 16, 1, 5] = x
    vc[pages[1, (length - 1) // 16].long(), (length - 1) % 16] = math.nan  # behind its last row
    _decode_check(gpu, q, kc, vc, pages, _ints(lens), seqs, lens)


def test_decode_cache_beyond_32_bit_offsets(gpu):
    """Rows whose byte offsets pass 2^32."""
    import torch

    gen, dt, page, Hkv, D = _gen(7), torch.bfloat16, 64, 8, 128
    n = (5 << 30) // (page * Hkv * D * 2)
    kc, vc = (torch.empty((n, page, Hkv, D), dtype=dt, device="cuda") for _ in range(2))
    lens = [300]
    pages = _ints([[n - 1 - 2 * i for i in range(5)]])
    k, v = (_randn(gen, 300, Hkv, D, dt=dt) for _ in range(2))
    assert gpu.kv_append(k, v, kc, vc, pages, _ints(list(range(300))), seqs=_ints([0] * 300)) is None
    q = _randn(gen, 1, 16, D, dt=dt)
    _decode_check(gpu, q, kc, vc, pages, _ints(lens), [(k, v)], lens)
    out = gpu.attend_prompt_paged(q, kc, vc, pages, _ints(lens), _ints([0, 1]))
    assert_attention(out, None, q, k, v, visible(1, 300, True, "cuda"), D ** -0.5)


def test_prompt_tokens_far_apart(gpu):
    """Packed rows 2 MB apart (offsets beyond 2^32), and rows so far apart that they are copied."""
    import torch

    gen, dt, n, D = _gen(24), torch.float16, 2504, 64
    room = torch.empty(n << 20, dtype=dt, device="cuda").view(n, 1 << 20)
    q, k, v = (room[:, i * 128:(i + 1) * 128].view(n, 2, D) for i in range(3))
    for t in (q, k, v):
        t.copy_(_randn(gen, n, 2, D, dt=dt))
    out = room[:, 512:640].view(n, 2, D)
    assert gpu.attend_prompt(q, k, v, _ints([0, 7, n]), out=out) is out
    for a, b in ((0, 7), (7, n)):
        assert_attention(out[a:b], None, q[a:b], k[a:b], v[a:b], visible(b - a, b - a, True, "cuda"), D ** -0.5)
    few = room.view(-1, 8 << 20)[:100, :384].view(100, 6, D)  # 16 MB apart
    q, k, v = few[:, :2], few[:, 2:4], few[:, 4:]
    got = gpu.attend_prompt(q, k, v, _ints([0, 100]))
    assert_attention(got, None, q, k, v, visible(100, 100, True, "cuda"), D ** -0.5)


def test_sequences_that_share_pages(gpu):
    """Two sequences with one prefix, their last pages their own: each reads the shared pages as its own."""
    import torch

    gen, dt, D, page = _gen(25), torch.bfloat16, 128, 16
    kc, vc, pages, seqs = paged(gen, [330, 50], page, 2, D, dt, width=21)
    k0, v0 = seqs[0]
    own = pages[1, :4].clone()
    pages[1] = pages[0]
    pages[1, 17:21] = own  # 272 shared rows, then the second's
    lens = [330, 272 + 50]
    seqs = [seqs[0], (torch.cat((k0[:272], seqs[1][0])), torch.cat((v0[:272], seqs[1][1])))]
    q = _randn(gen, 2, 8, D, dt=dt)
    _decode_check(gpu, q, kc, vc, pages, _ints(lens), seqs, lens)
    q = _randn(gen, 70, 8, D, dt=dt)
    out = gpu.attend_prompt_paged(q, kc, vc, pages, _ints(lens), _ints([0, 30, 70]))
    for b, (i, j) in enumerate(((0, 30), (30, 70))):
        assert_attention(out[i:j], None, q[i:j], *seqs[b], visible(j - i, lens[b], True, "cuda"), D ** -0.5)


def test_decode_strided_operands_and_given_buffers(gpu):
    import torch

    gen, dt = _gen(8), torch.bfloat16
    lens = [300, 17]
    kc, vc, pages, seqs = paged(gen, lens, 16, 2, 64, dt, order="heads")
    wide = torch.full((2, 30), -1, dtype=torch.int32, device="cuda")
    wide[:, :pages.shape[1]] = pages
    q = _randn(gen, 2, 9, 3, 64, dt=dt)[:, ::2, 1][:, :4]  # heads 384 apart
    room = torch.full((2, 6, 64), 3.0, dtype=dt, device="cuda")
    ws = torch.empty(gpu.attend_decode_workspace_size(2, 4, 2, 64, pages.shape[1], 16), dtype=torch.uint8, device="cuda")
    got = _decode_check(gpu, q, kc, vc, wide[:, :pages.shape[1]], _ints(lens), seqs, lens, out=room[:, 1:5], workspace=ws)
    assert got.data_ptr() == room[:, 1:5].data_ptr() and bool((room[:, 0] == 3).all()) and bool((room[:, 5] == 3).all())
    # Not 16-byte aligned: copied.
    odd = torch.empty(2 * 4 * 64 + 1, dtype=dt, device="cuda")[1:].view(2, 4, 64)
    odd.copy_(q)
    assert torch.equal(gpu.attend_decode(odd, kc, vc, pages, _ints(lens)), got)


@pytest.mark.parametrize("Hq,D,dtype", [(8, 128, "bf16"), (160, 128, "f16"), (24, 64, "f16"), (8, 256, "bf16")])
def test_decode_of_a_cache_larger_than_the_last_level_cache(gpu, Hq, D, dtype):
    """Page tables and pages of more than 256 MB: the rows' loads differ, the results do not."""
    import torch

    gen, dt, Hkv, page, lens = _gen(D + Hq), _dt(dtype), 8, 16, [300, 0, 2049, 1]
    n_pages = (256 << 20) // (4 * Hkv * D * page) + 1
    kc, vc, pages, seqs = paged(gen, lens, page, Hkv, D, dt, spare=n_pages, width=n_pages // 4 + 1)
    q, L = _randn(gen, 4, Hq, D, dt=dt), _ints(lens)
    out = _decode_check(gpu, q, kc, vc, pages, L, seqs, lens)
    used = -(-max(lens) // page)
    few = torch.cat((pages[:, :used], torch.full((4, pages.shape[1] // 2), -1, dtype=torch.int32, device="cuda")), 1)
    assert torch.equal(gpu.attend_decode(q, kc, vc, few, L), out)


@pytest.mark.parametrize("B,Hq,Hkv,D,most", [(64, 8, 4, 128, 1000), (43, 6, 6, 64, 641), (256, 40, 1, 72, 513)])
def test_decode_units_of_several_tiles_that_fill_the_chip(gpu, B, Hq, Hkv, D, most):
    import torch

    gen, dt = _gen(B), torch.bfloat16
    lens = [(97 * b + most) % (most + 1) for b in range(B)]
    lens[0] = most
    kc, vc, pages, seqs = paged(gen, lens, 16, Hkv, D, dt)
    q = _randn(gen, B, Hq, D, dt=dt)
    assert gpu.attend_decode_workspace_size(B, Hq, Hkv, D, pages.shape[1], 16) == 0
    _decode_check(gpu, q, kc, vc, pages, _ints(lens), seqs, lens)


@pytest.mark.parametrize("Hq,Hkv", [(1024, 1), (1024, 1024), (1024, 8), (1, 1)])
def test_most_and_fewest_heads(gpu, Hq, Hkv):
    import torch

    gen, dt, D, lens = _gen(Hq + Hkv), torch.float16, 8, [700, 3]
    kc, vc, pages, seqs = paged(gen, lens, 5, Hkv, D, dt)
    q = _randn(gen, 2, Hq, D, dt=dt)
    out = _decode_check(gpu, q, kc, vc, pages, _ints(lens), seqs, lens)
    k, v = (_randn(gen, 4, Hkv, D, dt=dt) for _ in range(2))
    pos = _ints([p - 1 for p in lens])  # over their last rows
    q2 = gpu.kv_append(k[:2], v[:2], kc, vc, pages, pos, q=q)
    assert torch.equal(q2, q)
    seqs = [(torch.cat((a[:-1], k[b:b + 1])), torch.cat((c[:-1], v[b:b + 1]))) for b, (a, c) in enumerate(seqs)]
    _decode_check(gpu, q, kc, vc, pages, _ints(lens), seqs, lens)
    lse = torch.empty((2, Hq), device="cuda")
    out = gpu.attend_prompt_paged(q, kc, vc, pages, _ints(lens), _ints([0, 1, 2]), lse=lse)
    for b, n in enumerate(lens):
        assert_attention(out[b:b + 1], lse[b:b + 1], q[b:b + 1], *seqs[b], visible(1, n, True, "cuda"), D ** -0.5)


# ---- numerics of both -----------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("score", [-9.0, -17.0])
def test_many_small_probabilities_keep_their_bits(gpu, dtype, score):
    """One key of weight 1 and value 0, 60000 of weight e^score and value 1: the result is all theirs.  e^-17 is 1.4 * 2^-25
    of the largest, below f16's smallest normal number."""
    import torch

    gen, dt, D, n, page = _gen(18), _dt(dtype), 64, 60001, 64
    kc, vc, pages, seqs = paged(gen, [n], page, 1, D, dt)
    k, v = seqs[0]
    k.zero_(), v.fill_(1.0)
    k[:, 0, 0] = score
    k[30, 0, 0], v[30] = 0.0, 0.0
    rows, at = pages[0].long(), torch.arange(n, device="cuda")
    kc[rows[at // page], at % page], vc[rows[at // page], at % page] = k, v
    q = torch.zeros((3, 2, D), dtype=dt, device="cuda")
    q[..., 0] = 1.0
    _decode_check(gpu, q[:1], kc, vc, pages, _ints([n]), seqs, [n], scale=1.0)
    seen = visible(3, n, True, "cuda")
    lse = torch.empty((3, 2), device="cuda")
    out = gpu.attend_prompt_paged(q, kc, vc, pages, _ints([n]), _ints([0, 3]), scale=1.0, lse=lse)
    assert_attention(out, lse, q, k, v, seen, 1.0)
    whole = gpu.attend_prompt(q, k, v, _ints([0, 3]), k_starts=_ints([0, n]), scale=1.0,
                              workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    assert_attention(whole, None, q, k, v, seen, 1.0)


def test_prompt_large_values_under_rising_scores(gpu):
    """Values of 2^115 under scores that rise by 0.05 a key (weights to 2^7 of the first tile's): the sums stay finite
    (200 weights of at most 1 are less than 2^8, the products' sums less than 2^123)."""
    import torch

    gen, dt, D, n = _gen(19), torch.bfloat16, 64, 200
    k, v = torch.zeros((n, 1, D), dtype=dt, device="cuda"), _randn(gen, n, 1, D, dt=dt).clamp(-4, 4) * 2.0 ** 113
    k[:, 0, 0] = torch.arange(n, device="cuda") * 0.05
    q = torch.zeros((n, 2, D), dtype=dt, device="cuda")
    q[..., 0] = 1.0
    out = gpu.attend_prompt(q, k, v, _ints([0, n]), scale=1.0)
    assert_attention(out, None, q, k, v, visible(n, n, True, "cuda"), 1.0)


# ---- prompt -------------------------------------------------------------------
def _prompt_check(gpu, gen, new, keys, Hq, Hkv, D, dt, causal, page=0, pad=0, by=2.0):
    import torch

    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    T = starts[-1] + pad
    q = _randn(gen, T, Hq, D, dt=dt, by=by)
    out = torch.full((T, Hq, D), 9.0, dtype=dt, device="cuda")
    lse = torch.full((T, Hq), 9.0, device="cuda")
    if page:
        kc, vc, pages, seqs = paged(gen, keys, page, Hkv, D, dt)
        gpu.attend_prompt_paged(q, kc, vc, pages, _ints(keys), _ints(starts), causal=causal, out=out, lse=lse)
    else:
        k_starts = [0]
        for m in keys:
            k_starts.append(k_starts[-1] + m)
        k, v = (_randn(gen, k_starts[-1] + pad, Hkv, D, dt=dt) for _ in range(2))
        seqs = [(k[a:b], v[a:b]) for a, b in zip(k_starts, k_starts[1:])]
        gpu.attend_prompt(q, k, v, _ints(starts), k_starts=_ints(k_starts), causal=causal, out=out, lse=lse)
    for b, (n, m) in enumerate(zip(new, keys)):
        r = slice(starts[b], starts[b + 1])
        assert_attention(out[r], lse[r], q[r], *seqs[b], visible(n, m, causal, "cuda"), D ** -0.5)
    assert bool((out[starts[-1]:] == 9).all()) and bool((lse[starts[-1]:] == 9).all())  # rows behind the last sequence


@pytest.mark.parametrize("Hq,Hkv,D,dtype", [
    (4, 1, 128, "bf16"), (2, 2, 64, "f16"), (3, 1, 256, "bf16"), (10, 2, 96, "f16"), (7, 1, 8, "bf16"), (33, 1, 40, "f16"),
    (2, 1, 168, "bf16"),
])
@pytest.mark.parametrize("new,keys", [
    ((1,), (1,)), ((0, 5, 0, 64, 1), (0, 5, 0, 64, 1)), ((130, 31, 257), (130, 31, 257)),
    ((3, 40, 1), (200, 41, 129)),       # keys in front of the new tokens
    ((70, 9, 4), (5, 0, 3)),            # fewer keys than queries: the first rows see none
])
@pytest.mark.parametrize("causal,page", [(True, 0), (False, 0), (True, 16), (True, 3), (False, 40)])
def test_prompt_matches_plain_attention(gpu, Hq, Hkv, D, dtype, new, keys, causal, page):
    _prompt_check(gpu, _gen(sum(new) + D), list(new), list(keys), Hq, Hkv, D, _dt(dtype), causal, page, pad=3)


@pytest.mark.parametrize("new,ahead,Hq,Hkv,D,page", [
    ((1500, 3, 700), 0, 8, 2, 128, 0), ((2000,), 0, 3, 3, 64, 0), ((600, 100), 3000, 8, 1, 128, 32), ((900,), 0, 2, 2, 256, 0),
    ((2100, 30), 0, 16, 16, 64, 0), ((1200, 1100, 1600), 0, 8, 8, 128, 0),
])
def test_prompt_long(gpu, new, ahead, Hq, Hkv, D, page):
    import torch

    _prompt_check(gpu, _gen(D), list(new), [n + ahead for n in new], Hq, Hkv, D, torch.bfloat16, True, page, by=4.0)


@pytest.mark.parametrize("new,ahead,Hq,Hkv,D,page,causal", [
    ((1,), 20001, 8, 1, 128, 64, True),              # one row tile, all the chip
    ((5, 64, 1, 0, 300), 4000, 6, 3, 64, 48, True),
    ((40, 3), 9000, 4, 2, 256, 16, False),
    ((2000, 10), 0, 2, 1, 96, 0, True),              # early rows see too little to be split
    ((1500,), 0, 4, 2, 128, 0, False),
    ((3, 700), 1500, 16, 1, 72, 7, True),
    ((700,), 0, 8, 1, 128, 0, True),                 # fewer units than CUs
    ((3, 20), 600, 4, 2, 64, 16, True),
    ((2100, 1000), 0, 16, 16, 64, 0, True),          # more units than CUs: the long sequence alone
    ((1400, 1100, 2200), 0, 8, 8, 128, 0, True),
    ((2050,), 0, 16, 16, 168, 0, True),
])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_prompt_split_over_the_keys(gpu, new, ahead, Hq, Hkv, D, page, causal, dtype):
    keys = [n + ahead // (1 + 2 * b) for b, n in enumerate(new)]
    assert gpu.attend_prompt_workspace_size(sum(new), len(new), Hq, Hkv, D, 0 if page else sum(keys), max(keys), 1) > 0
    _prompt_check(gpu, _gen(D), list(new), keys, Hq, Hkv, D, _dt(dtype), causal, page, by=3.0)


def test_prompt_workspace_given_short_or_whole(gpu):
    """Without its scratch a call takes each row tile in one workgroup: the same result to rounding."""
    import torch

    gen, dt, D = _gen(17), torch.bfloat16, 128
    kc, vc, pages, seqs = paged(gen, [9000], 64, 2, D, dt)
    q = _randn(gen, 70, 4, D, dt=dt)
    args = (q, kc, vc, pages, _ints([9000]), _ints([0, 70]))
    n = gpu.attend_prompt_workspace_size(70, 1, 4, 2, D, 0, pages.shape[1], 64)
    ws = torch.full((n,), 255, dtype=torch.uint8, device="cuda")
    want = gpu.attend_prompt_paged(*args)
    assert torch.equal(gpu.attend_prompt_paged(*args, workspace=ws), want)
    short = gpu.attend_prompt_paged(*args, workspace=ws[:n - 16])
    for got in (want, short):
        assert_attention(got, None, q, *seqs[0], visible(70, 9000, True, "cuda"), D ** -0.5)


def test_prompt_many_sequences(gpu):
    """More sequences than one look of a wave over `starts`."""
    import torch

    new = [(7 * i) % 5 for i in range(150)]
    _prompt_check(gpu, _gen(9), new, new, 4, 2, 64, torch.float16, True)
    _prompt_check(gpu, _gen(20), new, [n + 13 * (i % 9) for i, n in enumerate(new)], 4, 2, 64, torch.float16, True, page=16, pad=2)


@pytest.mark.parametrize("Hq,Hkv,D,dtype", [(8, 2, 128, "bf16"), (3, 1, 64, "f16"), (4, 4, 256, "bf16")])
def test_prompt_many_short_chunks_behind_cached_tokens(gpu, Hq, Hkv, D, dtype):
    """Row tiles that are partly rows, some of their sequences split over the keys."""
    new = [(5 * i) % 13 for i in range(40)]
    _prompt_check(gpu, _gen(26), new, [n + (97 * i) % 1500 for i, n in enumerate(new)], Hq, Hkv, D, _dt(dtype), True, page=16, pad=2)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_prompt_nan_and_infinity_do_not_reach_rows_that_do_not_see_them(gpu, D):
    import torch

    gen, dt, n = _gen(10), torch.bfloat16, 150
    q, k, v = (_randn(gen, n, 2, D, dt=dt) for _ in range(3))
    v[70, 0, 5], v[149, 1, 3], v[100, 0, 7] = math.nan, math.inf, -math.inf
    starts = _ints([0, n])
    out = gpu.attend_prompt(q, k, v, starts)
    assert_attention(out, None, q, k, v, visible(n, n, True, "cuda"), D ** -0.5)
    k[80, 1, 0] = math.nan  # a NaN score: the rows that see it are NaN, the others as they were
    got = gpu.attend_prompt(q, k, v, starts)
    assert torch.equal(got[:70], out[:70]) and torch.equal(got[70:80, 1], out[70:80, 1])
    assert torch.isnan(got[80:, 1]).all()


@pytest.mark.parametrize("page", [0, 16, 7])
@pytest.mark.parametrize("n,ahead,Hq,Hkv,D,dtype", [
    (150, 0, 6, 2, 64, "bf16"), (150, 40, 3, 1, 128, "f16"), (70, 1500, 6, 2, 128, "bf16"), (90, 1300, 5, 1, 256, "bf16"),
    (200, 900, 4, 4, 96, "f16"), (33, 700, 7, 1, 72, "bf16"),
])
def test_prompt_nan_and_infinity_among_cached_and_split_values(gpu, n, ahead, Hq, Hkv, D, dtype, page):
    """The same in the cache, for grouped heads and where the keys are split: in tiles that all rows see, that some do, and that
    only the last does."""
    import torch

    gen, dt, m = _gen(29), _dt(dtype), n + ahead
    q = _randn(gen, n, Hq, D, dt=dt)
    kc, vc, pages, seqs = paged(gen, [m], page or 64, Hkv, D, dt)
    k, v = seqs[0]
    split = gpu.attend_prompt_workspace_size(n, 1, Hq, Hkv, D, 0 if page else m, m, 1) > 0
    assert split == (m > 512)

    def check(at):
        v2 = v.clone()
        for i, (key, h, d, x) in enumerate(at):
            v2[key, h, d] = x
        starts = _ints([0, n])
        if page:
            rows = torch.arange(m, device="cuda")
            vc[pages[0].long()[rows // page], rows % page] = v2
        for ws in (None, torch.empty(16, dtype=torch.uint8, device="cuda")):  # with scratch, and in whole units
            lse = torch.empty((n, Hq), device="cuda")
            if page:
                out = gpu.attend_prompt_paged(q, kc, vc, pages, _ints([m]), starts, lse=lse, workspace=ws)
            else:
                out = gpu.attend_prompt(q, k, v2, starts, k_starts=_ints([0, m]), lse=lse, workspace=ws)
            assert_attention(out, lse, q, k, v2, visible(n, m, True, "cuda"), D ** -0.5)

    check([(m - 1, 0, 3, math.inf), (m - 1, Hkv - 1, D - 1, math.nan)])
    check([(ahead + n // 2, Hkv - 1, 0, math.nan), (ahead + 5, 0, D - 2, -math.inf), (ahead + 6, 0, D - 2, math.inf), (m - 2, 0, 1, math.nan)])
    if ahead:
        check([(ahead - 1, 0, 5, math.nan), (0, Hkv - 1, 6, math.inf)])


def test_prompt_masks_pages_that_do_not_exist(gpu):
    import torch

    gen, dt, page, D = _gen(11), torch.bfloat16, 16, 128
    kc, vc, pages, seqs = paged(gen, [200], page, 1, D, dt)
    pages[0, 4], pages[0, 0] = -2, kc.shape[0]
    q = _randn(gen, 90, 2, D, dt=dt)
    lse = torch.empty((90, 2), device="cuda")
    out = gpu.attend_prompt_paged(q, kc, vc, pages, _ints([200]), _ints([0, 90]), lse=lse)
    seen = visible(90, 200, True, "cuda").clone()
    seen[:, 64:80] = seen[:, :16] = False
    assert_attention(out, lse, q, *seqs[0], seen, D ** -0.5)


def test_prompt_fused_projection_views_and_bad_starts(gpu):
    import torch

    gen, dt, T, D = _gen(12), torch.float16, 200, 64
    qkv = _randn(gen, T, 8, D, dt=dt)
    q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
    out = gpu.attend_prompt(q, k, v, _ints([0, 60, 200]))
    for a, b in ((0, 60), (60, 200)):
        assert_attention(out[a:b], None, q[a:b], k[a:b], v[a:b], visible(b - a, b - a, True, "cuda"), D ** -0.5)
    # What passes the rows is cut off, what descends is empty (rows 40 .. 59 then belong to the third sequence too).
    room = torch.full_like(out, 9.0)
    gpu.attend_prompt(q, k, v, _ints([-3, 60, 40, 1000]), out=room)
    assert torch.equal(room[:40], out[:40])


@pytest.mark.parametrize("Hq,Hkv,D,page,dtype", [(8, 2, 128, 16, "bf16"), (6, 3, 72, 5, "f16"), (4, 2, 256, 8, "bf16"), (5, 1, 64, 24, "f16")])
def test_keys_and_values_in_caches_of_other_strides(gpu, Hq, Hkv, D, page, dtype):
    """Keys by rows, values by heads, each a part of something wider."""
    import torch

    gen, dt, lens = _gen(31), _dt(dtype), [70, 1100, 0, 1]
    kc, vc, pages, seqs = paged(gen, lens, page, Hkv, D, dt)
    wide = torch.full((kc.shape[0], 2, page, Hkv + 1, D + 8), math.nan, dtype=dt, device="cuda")
    k2 = wide[:, 1, :, 1:, 8:]
    k2.copy_(kc)
    v2 = torch.full((kc.shape[0], Hkv, 3, page, D), math.nan, dtype=dt, device="cuda")[:, :, 1].transpose(1, 2)
    v2.copy_(vc)
    q = _randn(gen, 4, Hq, D, dt=dt)
    _decode_check(gpu, q, k2, v2, pages, _ints(lens), seqs, lens)
    starts = [0, 33, 93, 95, 96]
    q = _randn(gen, 96, Hq, D, dt=dt)
    lse = torch.empty((96, Hq), device="cuda")
    out = gpu.attend_prompt_paged(q, k2, v2, pages, _ints(lens), _ints(starts), lse=lse)
    for b, n in enumerate(lens):
        r = slice(starts[b], starts[b + 1])
        assert_attention(out[r], lse[r], q[r], *seqs[b], visible(starts[b + 1] - starts[b], n, True, "cuda"), D ** -0.5)
    k, v = (_randn(gen, 3, Hkv, D, dt=dt) for _ in range(2))
    before = wide.clone()
    gpu.kv_append(k, v, k2, v2, pages, _ints([3, 69, 1099]), seqs=_ints([0, 0, 1]))
    for t, (b, p) in enumerate(((0, 3), (0, 69), (1, 1099))):
        at = int(pages[b, p // page]), p % page
        assert torch.equal(k2[at], k[t]) and torch.equal(v2[at], v[t])
        before[at[0], 1, at[1], 1:, 8:] = k[t]
    assert torch.equal(wide.view(torch.int16), before.view(torch.int16))


def test_prompt_broadcast_operands(gpu):
    """Heads and tokens of one place, among the operands that are read."""
    import torch

    gen, dt, T, D = _gen(32), torch.bfloat16, 140, 64
    q, k, v = _randn(gen, 1, 4, D, dt=dt).expand(T, 4, D), _randn(gen, T, 1, D, dt=dt).expand(T, 2, D), _randn(gen, T, 1, D, dt=dt).expand(T, 2, D)
    out = gpu.attend_prompt(q, k, v, _ints([0, 100, T]))
    for a, b in ((0, 100), (100, T)):
        assert_attention(out[a:b], None, q[a:b], k[a:b], v[a:b], visible(b - a, b - a, True, "cuda"), D ** -0.5)
    kc, vc, pages, _ = paged(gen, [T], 16, 2, D, dt)
    gpu.kv_append(k, v, kc, vc, pages, _ints(list(range(T))), seqs=_ints([0] * T))
    assert torch.equal(gpu.attend_prompt_paged(q, kc, vc, pages, _ints([T]), _ints([0, T]))[:100], out[:100])
    one = kc[:, :, :1].expand(-1, -1, 2, -1), vc[:, :, :1].expand(-1, -1, 2, -1)
    L = _ints([T])
    assert torch.equal(gpu.attend_decode(q[:1], *one, pages, L), gpu.attend_decode(q[:1], kc, vc, pages, L))


@pytest.mark.parametrize("B", [63, 64, 65])
@pytest.mark.parametrize("Hq,Hkv,D", [(2, 1, 64), (4, 2, 256)])
def test_prompt_one_long_sequence_among_as_many_as_a_wave_has_lanes(gpu, B, Hq, Hkv, D):
    new = [1 + (11 * i) % 7 for i in range(B)]
    new[B - 2] = 90
    keys = [n + (B - i) % 40 for i, n in enumerate(new)]
    keys[B - 2] = 2600
    split = gpu.attend_prompt_workspace_size(sum(new), B, Hq, Hkv, D, 0, 2600, 1) > 0
    assert split == (B <= 64)
    _prompt_check(gpu, _gen(33), new, keys, Hq, Hkv, D, _dt("bf16"), True, page=16, pad=1)
    _prompt_check(gpu, _gen(34), new, keys, Hq, Hkv, D, _dt("f16"), True, pad=1)


# ---- streams, graphs ------------------------------------------------------------
def test_calls_on_another_stream(gpu):
    import torch

    gen, dt = _gen(13), torch.bfloat16
    lens = [500, 900]
    kc, vc, pages, _ = paged(gen, lens, 16, 2, 128, dt)
    q, L = _randn(gen, 2, 8, 128, dt=dt), _ints(lens)
    want = gpu.attend_decode(q, kc, vc, pages, L)
    wide = _randn(gen, 40, 8, 128, dt=dt)
    want_p = gpu.attend_prompt_paged(wide, kc, vc, pages, L, _ints([0, 10, 40]))
    starts = _ints([0, 10, 40])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = gpu.attend_decode(q, kc, vc, pages, L, stream=side)
    got_p = gpu.attend_prompt_paged(wide, kc, vc, pages, L, starts, stream=side)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(got_p, want_p)


def test_stream_of_another_device_is_refused(gpu):
    import torch

    side = torch.cuda.Stream()
    kc = torch.zeros((2, 4, 1, 8), dtype=torch.float16)
    q, pages, one = torch.zeros((1, 1, 8), dtype=torch.float16), torch.zeros((1, 2), dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    for call in (lambda: gpu.kv_append(q, q, kc, kc, pages, one, stream=side), lambda: gpu.attend_decode(q, kc, kc, pages, one, stream=side),
                 lambda: gpu.attend_prompt(q, q, q, one, stream=side), lambda: gpu.attend_prompt_paged(q, kc, kc, pages, one, one, stream=side)):
        with pytest.raises(ValueError, match="stream"):
            call()


def test_captured_step_replays(gpu):
    """Append, attend and count in one graph, replayed with the host's own work between; two graphs in turn."""
    import torch

    gen, dt, B, Hq, Hkv, D, page = _gen(14), torch.bfloat16, 3, 8, 2, 64, 16
    rope = gpu.rope_table(200, D)
    first = [5, 90, 0]

    def make():
        g = _gen(15)
        kc, vc, pages, _ = paged(g, [160] * B, page, Hkv, D, dt)
        return dict(kc=kc, vc=vc, pages=pages, pos=_ints(first), x=_randn(g, B, Hq + 2 * Hkv, D, dt=dt),
                    out=torch.empty((B, Hq, D), dtype=dt, device="cuda"))

    def step(s):
        q, k, v = s["x"][:, :Hq], s["x"][:, Hq:Hq + Hkv], s["x"][:, Hq + Hkv:]
        r = gpu.kv_append(k, v, s["kc"], s["vc"], s["pages"], s["pos"], q=q, rope=rope)
        gpu.attend_decode(r, s["kc"], s["vc"], s["pages"], s["pos"] + 1, out=s["out"])
        s["pos"].add_(1)

    eager, a, b = make(), make(), make()
    for s in (eager, a, b):
        s["kc"].zero_(), s["vc"].zero_()
    graphs = []
    for s in (a, b):
        step(s)  # warm
        s["pos"].copy_(_ints(first))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(s)
        graphs.append(g)
    for i in range(6):
        x = _randn(gen, B, Hq + 2 * Hkv, D, dt=dt)
        for s in (eager, a, b):
            s["x"].copy_(x)
        step(eager)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(a["out"], eager["out"]) and torch.equal(b["out"], eager["out"]), i
        assert torch.equal(a["pos"], eager["pos"])
        torch.randn((1000, 1000), device="cuda") @ torch.randn((1000, 1000), device="cuda")


def test_captured_prompts_replay_over_other_lengths(gpu):
    """A chunk of two prompts, split over the keys, in a graph: replayed as the cache grows and the chunk divides otherwise."""
    import torch

    gen, dt, D, page = _gen(21), torch.float16, 128, 16
    kc, vc, pages, _ = paged(gen, [6000, 4000], page, 2, D, dt)
    q, starts, lengths = _randn(gen, 100, 8, D, dt=dt), _ints([0, 60, 100]), _ints([5000, 40])
    out, lse = torch.zeros_like(q), torch.zeros((100, 8), device="cuda")
    call = lambda: gpu.attend_prompt_paged(q, kc, vc, pages, lengths, starts, out=out, lse=lse)
    call()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for new, keys in (([0, 60, 100], [5000, 40]), ([0, 1, 100], [6000, 4000]), ([0, 0, 90], [0, 3333]), ([5, 100, 100], [700, 0])):
        starts.copy_(_ints(new)), lengths.copy_(_ints(keys)), q.copy_(_randn(gen, 100, 8, D, dt=dt))
        out.fill_(9.0), lse.fill_(9.0)
        g.replay()
        torch.cuda.synchronize()
        got = out.clone(), lse.clone()
        out.fill_(9.0), lse.fill_(9.0)
        call()
        assert torch.equal(got[0], out) and torch.equal(got[1], lse)
        torch.randn((1000, 1000), device="cuda") @ torch.randn((1000, 1000), device="cuda")


def test_two_calls_at_once(gpu):
    """Calls on two streams, each with scratch of its own, as the calls take it when none is given."""
    import torch

    gen, dt, D, lens = _gen(22), torch.bfloat16, 128, [9000, 100]
    kc, vc, pages, _ = paged(gen, lens, 16, 2, D, dt)
    L, starts = _ints(lens), _ints([0, 30, 50])
    q = [_randn(gen, 2, 16, D, dt=dt) for _ in range(2)]
    p = [_randn(gen, 50, 16, D, dt=dt) for _ in range(2)]
    want = [(gpu.attend_decode(a, kc, vc, pages, L), gpu.attend_prompt_paged(b, kc, vc, pages, L, starts)) for a, b in zip(q, p)]
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(sides):
            got[i].append((gpu.attend_decode(q[i], kc, vc, pages, L, stream=s),
                           gpu.attend_prompt_paged(p[i], kc, vc, pages, L, starts, stream=s)))
    torch.cuda.synchronize()
    for i in range(2):
        for a, b in got[i]:
            assert torch.equal(a, want[i][0]) and torch.equal(b, want[i][1])


def test_operands_that_want_gradients_are_refused(gpu):
    import torch

    gen, dt = _gen(23), torch.bfloat16
    kc, vc, pages, _ = paged(gen, [20], 16, 1, 32, dt)
    q, k, v = (_randn(gen, 1, 1, 32, dt=dt) for _ in range(3))
    L, starts = _ints([20]), _ints([0, 1])
    calls = (lambda q, k, v, kc, vc: gpu.kv_append(k, v, kc, vc, pages, _ints([3]), q=q),
             lambda q, k, v, kc, vc: gpu.attend_prompt(q, k, v, starts),
             lambda q, k, v, kc, vc: gpu.attend_prompt_paged(q, kc, vc, pages, L, starts),
             lambda q, k, v, kc, vc: gpu.attend_decode(q, kc, vc, pages, L))
    used = ((0, 1, 2, 3, 4), (0, 1, 2), (0, 3, 4), (0, 3, 4))
    for call, which in zip(calls, used):
        for i in which:
            args = [q, k, v, kc, vc]
            args[i] = args[i].clone().requires_grad_()
            with pytest.raises(RuntimeError, match="no_grad"):
                call(*args)
            with torch.no_grad():
                call(*args)


def test_operands_with_tangents_are_refused(gpu):
    """Forward-mode derivatives would be dropped: operands that carry one are refused, lse and out among them."""
    import torch
    import torch.autograd.forward_ad as fwd

    gen, dt = _gen(27), torch.bfloat16
    kc, vc, pages, _ = paged(gen, [20], 16, 1, 32, dt)
    q, k, v, out = (_randn(gen, 1, 1, 32, dt=dt) for _ in range(4))
    rope, lse, L, starts = gpu.rope_table(20, 32), torch.zeros((1, 1), device="cuda"), _ints([20]), _ints([0, 1])
    calls = (lambda q, k, v, kc, vc, out, lse, rope: gpu.kv_append(k, v, kc, vc, pages, _ints([3]), q=q, q_out=out, rope=rope),
             lambda q, k, v, kc, vc, out, lse, rope: gpu.attend_prompt(q, k, v, starts, out=out, lse=lse),
             lambda q, k, v, kc, vc, out, lse, rope: gpu.attend_prompt_paged(q, kc, vc, pages, L, starts, out=out, lse=lse),
             lambda q, k, v, kc, vc, out, lse, rope: gpu.attend_decode(q, kc, vc, pages, L, out=out, lse=lse))
    used = ((0, 1, 2, 3, 4, 5, 7), (0, 1, 2, 5, 6), (0, 3, 4, 5, 6), (0, 3, 4, 5, 6))
    for call, which in zip(calls, used):
        for i in which:
            args = [q, k, v, kc, vc, out, lse, rope]
            with fwd.dual_level():
                args[i] = fwd.make_dual(args[i], torch.ones_like(args[i]))
                with pytest.raises(RuntimeError, match="derivative"):
                    call(*args)
                with torch.no_grad(), pytest.raises(RuntimeError, match="derivative"):  # which does not stop tangents
                    call(*args)
            call(q, k, v, kc, vc, out, lse, rope)
    with pytest.raises(RuntimeError, match="no_grad"):
        gpu.attend_decode(q, kc, vc, pages, L, lse=lse.clone().requires_grad_())


def test_what_is_written_counts_as_changed(gpu):
    """A buffer that autograd saved and a call then fills is noticed at the backward pass, as with torch's own in-place operations."""
    import torch

    gen, dt = _gen(28), torch.bfloat16
    kc, vc, pages, _ = paged(gen, [20], 16, 1, 32, dt)
    q, k, v, out, q_out = (_randn(gen, 1, 1, 32, dt=dt) for _ in range(5))
    lse, L, starts = torch.zeros((1, 1), device="cuda"), _ints([20]), _ints([0, 1])
    calls = ((lambda: gpu.kv_append(k, v, kc, vc, pages, _ints([3]), q=q, q_out=q_out), (kc, vc, q_out)),
             (lambda: gpu.attend_prompt(q, k, v, starts, out=out, lse=lse), (out, lse)),
             (lambda: gpu.attend_prompt_paged(q, kc, vc, pages, L, starts, out=out, lse=lse), (out, lse)),
             (lambda: gpu.attend_decode(q, kc, vc, pages, L, out=out, lse=lse), (out, lse)))
    read = (q, k, v, pages, L, starts)
    for call, written in calls:
        before = [t._version for t in (*written, *read)]
        call()
        assert [t._version for t in written] == [n + 1 for n in before[:len(written)]]
        assert [t._version for t in read] == before[len(written):]
    w = torch.ones(32, dtype=dt, device="cuda", requires_grad=True)
    y = (w * out).sum()
    gpu.attend_decode(q, kc, vc, pages, L, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        mine = torch.empty_like(out)
        gpu.attend_decode(q, kc, vc, pages, L, out=mine)
    gpu.attend_decode(q, kc, vc, pages, L, out=mine)  # inference tensors have no counter
    assert torch.equal(mine, out)


def _refusal_operands():
    import torch

    dt = torch.bfloat16
    t = lambda *shape, dt=dt: torch.zeros(shape, dtype=dt, device="cuda")
    return dict(q=t(3, 4, 64), k=t(3, 2, 64), v=t(3, 2, 64), kc=t(4, 8, 2, 64), vc=t(4, 8, 2, 64), pages=t(3, 2, dt=torch.int32),
                ints=t(3, dt=torch.int32), starts=t(4, dt=torch.int32))


REFUSED = [  # which operand, what it becomes
    ("q", lambda t, o: t[0], ValueError), ("q", lambda t, o: t.half(), TypeError), ("q", lambda t, o: t.float(), TypeError),
    ("q", lambda t, o: t[..., :56], ValueError), ("q", lambda t, o: t.cpu(), ValueError),
    ("kc", lambda t, o: t[0], ValueError), ("kc", lambda t, o: t.half(), TypeError), ("kc", lambda t, o: t[:2], ValueError),
    ("vc", lambda t, o: t.half(), TypeError), ("vc", lambda t, o: t.cpu(), ValueError),
    ("vc", lambda t, o: t.transpose(2, 3).contiguous().transpose(2, 3), ValueError),
    ("kc", lambda t, o: t.expand(4, 8, 2, 64)[..., ::2], ValueError),
    ("pages", lambda t, o: t.long(), ValueError), ("pages", lambda t, o: t[0], ValueError), ("pages", lambda t, o: t.cpu(), ValueError),
    ("pages", lambda t, o: t.T.contiguous().T, ValueError),
    ("ints", lambda t, o: t.long(), ValueError), ("ints", lambda t, o: t[:2], ValueError), ("ints", lambda t, o: t.cpu(), ValueError),
]


@pytest.mark.parametrize("at", range(len(REFUSED)))
def test_operands_that_do_not_fit_are_refused(gpu, at):
    which, change, error = REFUSED[at]
    calls = (lambda q, k, v, kc, vc, pages, ints, starts: gpu.kv_append(k, v, kc, vc, pages, ints, q=q),
             lambda q, k, v, kc, vc, pages, ints, starts: gpu.attend_decode(q, kc, vc, pages, ints),
             lambda q, k, v, kc, vc, pages, ints, starts: gpu.attend_prompt_paged(q, kc, vc, pages, ints, starts))
    for call in calls:
        o = _refusal_operands()
        call(**o)
        o[which] = change(o[which], o)
        with pytest.raises(error):
            call(**o)


def test_options_that_do_not_fit_are_refused(gpu):
    import torch

    o = _refusal_operands()
    q, k, v, kc, vc, pages, ints, starts = o.values()
    decode = lambda **kw: gpu.attend_decode(q, kc, vc, pages, ints, **kw)
    prompt = lambda **kw: gpu.attend_prompt(q, k, v, starts, **kw)
    paged_ = lambda **kw: gpu.attend_prompt_paged(q, kc, vc, pages, ints, starts, **kw)
    for call in (decode, prompt, paged_):
        for scale in (0.0, -1.0, math.inf, math.nan):
            with pytest.raises(ValueError, match="scale"):
                call(scale=scale)
        with pytest.raises(TypeError):
            call(scale="x")
        for out in (q[:2], q.half(), q.cpu(), torch.zeros((3, 4, 128), dtype=q.dtype, device="cuda")[..., ::2],
                    torch.zeros(3 * 4 * 64 + 1, dtype=q.dtype, device="cuda")[1:].view(3, 4, 64)):
            with pytest.raises(ValueError, match="out"):
                call(out=out)
        with pytest.raises(TypeError, match="out"):
            call(out=3)
        with pytest.raises(gpu.LatentError):
            call(out=torch.zeros((3, 1, 64), dtype=q.dtype, device="cuda").expand(3, 4, 64))  # heads of one place
        for lse in (torch.zeros((3, 3), device="cuda"), torch.zeros((3, 4)), torch.zeros((4, 3), device="cuda").T,
                    torch.zeros((3, 4), dtype=torch.float64, device="cuda")):
            with pytest.raises(ValueError, match="lse"):
                call(lse=lse)
        with pytest.raises(ValueError, match="workspace"):
            call(workspace=torch.zeros(64, dtype=torch.uint8))
        with pytest.raises(gpu.LatentError):
            call(workspace=None, scale=1.0, out=torch.zeros((3, 4, 64 + 8), dtype=q.dtype, device="cuda")[..., :64][:, :1].expand(3, 4, 64))
    for bad in (starts[:0], starts.view(2, 2), starts.long(), starts.cpu(), torch.zeros(2, dtype=torch.int32, device="cuda")):
        with pytest.raises(ValueError):
            gpu.attend_prompt_paged(q, kc, vc, pages, ints, bad)
    for bad in (starts[:0], starts.view(2, 2), starts.long(), starts.cpu()):
        with pytest.raises(ValueError):
            gpu.attend_prompt(q, k, v, bad)
    with pytest.raises(ValueError, match="k_starts"):
        gpu.attend_prompt(q, k[:2], v[:2], starts)
    with pytest.raises(ValueError, match="k_starts"):
        gpu.attend_prompt(q, k[:2], v[:2], starts, k_starts=starts[:3])
    with pytest.raises(ValueError):
        gpu.attend_prompt(q[:, :3], k, v, starts)  # 3 heads over 2
    with pytest.raises(ValueError):
        gpu.attend_prompt(q, k, v[:2], starts)
    append = lambda **kw: gpu.kv_append(k, v, kc, vc, pages, ints, **kw)
    for rope in (torch.zeros((4, 2, 33), device="cuda"), torch.zeros((4, 2, 0), device="cuda"), torch.zeros((4, 32), device="cuda"),
                 torch.zeros((4, 2, 32)), torch.zeros((4, 2, 32), device="cuda").half()):
        with pytest.raises(ValueError, match="rope"):
            append(rope=rope)
    with pytest.raises(ValueError, match="q_out"):
        append(q_out=q)
    with pytest.raises(ValueError, match="seqs"):
        append(seqs=ints[:2])
    with pytest.raises(ValueError, match="seqs"):
        gpu.kv_append(k, v, kc, vc, pages[:2], ints)
    with pytest.raises(gpu.LatentError):  # pages of one place
        gpu.kv_append(k, v, kc[:1].expand(4, 8, 2, 64), vc, pages, ints)
    with pytest.raises(gpu.LatentError):  # heads of 20
        gpu.attend_prompt(q[..., :20].contiguous(), k[..., :20].contiguous(), v[..., :20].contiguous(), starts)


# ---- a run of them together -----------------------------------------------------
def test_prompt_then_tokens_equal_one_prompt(gpu):
    """Prompts appended in chunks and continued token by token see what one packed causal pass sees."""
    import torch

    gen, dt, Hq, Hkv, D, page = _gen(16), torch.bfloat16, 8, 2, 64, 16
    lens, B = [133, 37, 64], 3
    rope = gpu.rope_table(200, D)
    kc, vc, pages, _ = paged(gen, lens, page, Hkv, D, dt)
    q, k, v = ([_randn(gen, n, h, D, dt=dt) for n in lens] for h in (Hq, Hkv, Hkv))
    turned = []
    # The oracle's rows: rotated operands as the kernel rounds them.
    out = [torch.empty((n, Hq, D), dtype=dt, device="cuda") for n in lens]
    done = [0] * B
    rot_q = [[] for _ in range(B)]
    for chunk in ([60, 10, 1], [70, 25, 62], [1, 1, 0], [1, 1, 1], [1, 0, 0]):
        T = sum(chunk)
        take = [slice(done[b], done[b] + chunk[b]) for b in range(B)]
        qq, kk, vv = (torch.cat([x[b][take[b]] for b in range(B)]) for x in (q, k, v))
        seqs = _ints([b for b in range(B) for _ in range(chunk[b])])
        pos = _ints([p for b in range(B) for p in range(done[b], done[b] + chunk[b])])
        r = gpu.kv_append(kk, vv, kc, vc, pages, pos, seqs=seqs, q=qq, rope=rope)
        done = [d + c for d, c in zip(done, chunk)]
        starts = [0]
        for c in chunk:
            starts.append(starts[-1] + c)
        if max(chunk) == 1:  # the single-token form, sequences without a new token padded
            wide = torch.zeros((B, Hq, D), dtype=dt, device="cuda")
            wide[seqs.long()] = r
            got = gpu.attend_decode(wide, kc, vc, pages, _ints([d if c else 0 for d, c in zip(done, chunk)]))[seqs.long()]
        else:
            got = gpu.attend_prompt_paged(r, kc, vc, pages, _ints(done), _ints(starts))
        for b in range(B):
            out[b][take[b]] = got[starts[b]:starts[b + 1]]
            rot_q[b].append(r[starts[b]:starts[b + 1]])
    for b, n in enumerate(lens):
        p = torch.arange(n, device="cuda")
        rows = pages[b].long()[p // page]
        turned.append(kc[rows, p % page])
        assert done[b] == n
        assert_attention(out[b], None, torch.cat(rot_q[b]), turned[b], v[b], visible(n, n, True, "cuda"), D ** -0.5)
