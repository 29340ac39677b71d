"""8-bit paged caches on the GPU: written, read back, attended to, against plain torch operations (to the bit) and 64 bits."""

import math

import pytest
import torch

from tests._attention import assert_attention, visible
from tests._cache8 import CODES, bits, empty_cache, paged8, put, quantise, take, values

pytestmark = pytest.mark.gpu
DT = {"f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def la(gpu):
    return gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def rotated(x, table, positions, interleaved):
    """fp32, products and sums rounded one by one."""
    x = x.float()
    rot = 2 * table.shape[2]
    cos, sin = (t[:, None, :] for t in table[positions.long()].unbind(1))
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    first, second = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((first, second), -1).flatten(-2) if interleaved else torch.cat((first, second), -1)
    return torch.cat((turned, x[..., rot:]), -1)


# ---- append, read --------------------------------------------------------------
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("D,rot,interleaved,Hq,Hkv,T,page,order", [
    (128, 128, False, 4, 2, 5, 16, "rows"), (64, 32, True, 7, 1, 37, 8, "rows"), (80, 80, False, 2, 2, 3, 24, "heads"), (96, 32, False, 0, 3, 9, 16, "rows"),
    (256, 128, True, 2, 2, 11, 16, "heads"), (16, 16, False, 1, 1, 1, 8, "rows"), (128, 20, False, 4, 2, 6, 16, "rows"),
    (112, 102, True, 3, 3, 6, 16, "rows"), (128, 0, False, 4, 2, 6, 16, "rows"), (128, 128, False, 16, 8, 700, 32, "rows"), (256, 256, False, 8, 8, 300, 16, "rows"),
    (64, 64, True, 14, 2, 900, 64, "rows"), (48, 12, False, 12, 4, 801, 8, "rows")])
def test_append_and_read_back(la, code, dt, D, rot, interleaved, Hq, Hkv, T, page, order):
    g, dt, code = gen(T + D), DT[dt], CODES[code]
    B, far = 3, 8 * T + 50
    width = -(-far // page)
    n = B * width + 2
    pages = torch.randperm(n, generator=g, device="cuda")[:B * width].int().view(B, width)
    seqs = torch.randint(0, B, (T,), generator=g, device="cuda").int()
    positions = torch.randperm(far, generator=g, device="cuda")[:T].int()
    kc, ks = empty_cache(n, page, Hkv, D, code, order=order)
    vc, vs = empty_cache(n, page, Hkv, D, code, order=order)
    want = [t.clone() for t in (bits(kc), bits(vc), ks, vs)]
    qkv = (torch.randn((T, Hq + 2 * Hkv, D), generator=g, device="cuda") * torch.exp2(torch.randn((T, 1, 1), generator=g, device="cuda"))).to(dt)
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    table = la.rope_table(far, rot) if rot else None
    got = la.kv_append(k, v, kc, vc, pages, positions, seqs=seqs, q=q if Hq else None, rope=table, interleaved=interleaved, k_scale=ks, v_scale=vs)
    rows, at = pages[seqs.long(), positions.long() // page].long(), positions.long() % page
    stored = []
    for x, c, s in ((rotated(k, table, positions, interleaved) if rot else k, want[0], want[2]), (v, want[1], want[3])):
        codes, scale = quantise(x, code)
        c[rows, at] = bits(codes)
        s[rows, :, at] = scale
        stored.append((codes.float() * scale[..., None]).to(dt))
    for a, b in zip((bits(kc), bits(vc), ks, vs), want):  # what was not named is as it was
        assert torch.equal(a.view(torch.int32 if a.dtype == torch.float32 else a.dtype), b.view(torch.int32 if b.dtype == torch.float32 else b.dtype))
    if Hq:
        exact = rotated(q.double(), table.double(), positions, interleaved).double() if rot else q.double()
        # products and a sum in fp32 (2^-24 of each product), one rounding
        size = q.double().abs().amax(-1, keepdim=True) * 2
        assert bool(((got.double() - exact).abs() <= size * 2 * 3 * 2.0 ** -24 + exact.abs() * torch.finfo(dt).eps / 2 + 2.0 ** -24).all())
    kr, vr = la.kv_read(kc, vc, pages, positions, seqs=seqs, k_scale=ks, v_scale=vs, dtype=dt)
    assert torch.equal(kr, stored[0]) and torch.equal(vr, stored[1])


@pytest.mark.parametrize("code", CODES)
def test_what_does_not_exist_is_left_out_and_reads_as_zeros(la, code):
    g, code = gen(5), CODES[code]
    kc, ks = empty_cache(6, 8, 2, 32, code)
    vc, vs = empty_cache(6, 8, 2, 32, code)
    pages = ints([[0, 1, -1], [2, 6, 3]])
    #          fine  page -1  page 6  behind  negative  sequence 2  sequence -1  behind the rope table
    positions = ints([9, 17, 9, 24, -1, 0, 0, 21])
    seqs = ints([0, 0, 1, 1, 0, 2, -1, 1])
    k, v, q = (torch.randn((8, h, 32), generator=g, device="cuda").half() for h in (2, 2, 4))
    before = [bits(kc).clone(), bits(vc).clone()]
    out = torch.full_like(q, 7.0)
    la.kv_append(k, v, kc, vc, pages, positions, seqs=seqs, q=q, rope=la.rope_table(21, 32), q_out=out, k_scale=ks, v_scale=vs)
    for c, was, s in ((kc, before[0], ks), (vc, before[1], vs)):
        changed = (bits(c) != was).any(-1).any(-1)
        assert changed.sum() == 1 and changed[1, 1] and torch.isfinite(s).sum() == 2 and torch.isfinite(s[1, :, 1]).all()
    assert torch.equal((out == 7.0).all(-1).all(-1), torch.tensor([0, 0, 0, 1, 1, 0, 0, 1], device="cuda").bool())
    kr, vr = la.kv_read(kc, vc, pages, positions, seqs=seqs, k_scale=ks, v_scale=vs, dtype=torch.float16)
    for r, c, s in ((kr, kc, ks), (vr, vc, vs)):
        assert torch.equal(r[0], values(take(c, 1, 1), s[1, :, 1]).half())
        # the last exists, unwritten: a NaN's scale
        assert bool((r[1:7] == 0).all()) and bool(torch.isnan(r[7]).all())


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dt", DT)
def test_rows_of_zeros_tiny_rows_and_rows_that_are_not_finite(la, code, dt):
    code, dt = CODES[code], DT[dt]
    D = 48
    rows = torch.zeros((7, 1, D), dtype=dt, device="cuda")
    rows[1] = torch.finfo(dt).smallest_normal
    rows[2] = torch.finfo(dt).tiny * 2.0 ** -5  # not a normal number
    rows[3] = torch.linspace(-1, 1, D, device="cuda").to(dt) * torch.finfo(dt).max
    rows[4, 0, 5], rows[5, 0, 47], rows[6, 0, 0] = math.inf, math.nan, -math.inf
    kc, ks = empty_cache(1, 8, 1, D, code)
    vc, vs = empty_cache(1, 8, 1, D, code)
    seqs, positions = ints([0] * 7), ints(range(7))
    la.kv_append(rows, rows, kc, vc, ints([[0]]), positions, seqs=seqs, k_scale=ks, v_scale=vs)
    codes, scale = quantise(rows, code)
    for c, s in ((kc, ks), (vc, vs)):
        assert torch.equal(bits(c)[0, :7, 0], bits(codes)[:, 0]) and torch.equal(s[0, 0, :4], scale[:4, 0]) and bool(torch.isnan(s[0, 0, 4:7]).all())
    k, v = la.kv_read(kc, vc, ints([[0]]), positions, seqs=seqs, k_scale=ks, v_scale=vs, dtype=dt)
    assert bool(torch.isfinite(k[:4]).all()) and bool(torch.isnan(k[4:]).all()) and bool(torch.isnan(v[4:]).all())


@pytest.mark.parametrize("dt", DT)
def test_a_16_bit_cache_is_read_as_it_is(la, dt):
    g, dt = gen(9), DT[dt]
    kc, vc = (torch.randn((5, 3, 2, 72), generator=g, device="cuda").to(dt) for _ in range(2))  # any page size, any D of the cache
    pages, positions, seqs = ints([[4, 0], [2, 9]]), ints([0, 5, 2, 3, 6]), ints([0, 0, 1, 1, 0])
    k, v = la.kv_read(kc, vc, pages, positions, seqs=seqs)
    for r, c in ((k, kc), (v, vc)):
        assert r.dtype == dt and torch.equal(r[:3], torch.stack((c[4, 0], c[0, 2], c[2, 2]))) and bool((r[3:] == 0).all())
    assert torch.equal(la.kv_read(kc, vc, pages, positions, seqs=seqs, dtype=dt)[0], k)


# ---- attention -----------------------------------------------------------------
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("lengths,Hkv,G,D,page,width,order", [
    ([1], 1, 1, 16, 8, None, "rows"), ([0, 7, 8, 9, 31, 32, 33], 2, 4, 64, 8, None, "rows"), ([127, 128, 129, 0, 500], 2, 3, 128, 16, None, "rows"),
    ([300, 1], 1, 17, 128, 48, None, "heads"), ([200, 77], 2, 20, 64, 16, None, "rows"), ([700], 1, 33, 80, 16, None, "rows"),
    ([40, 900], 2, 2, 96, 24, 200, "rows"), ([650, 3], 2, 16, 256, 16, 80, "heads"), ([513, 12], 1, 18, 192, 16, None, "rows"), ([5000, 0, 1, 1200], 2, 8, 128, 16, None, "rows"),
    ([3000], 1, 8, 256, 64, None, "rows")])
def test_decode(la, code, dt, lengths, Hkv, G, D, page, width, order):
    g, dt = gen(sum(lengths) + D), DT[dt]
    kc, vc, ks, vs, pages, seqs = paged8(g, lengths, page, Hkv, D, dt, CODES[code], width=width, order=order)
    q = (torch.randn((len(lengths), Hkv * G, D), generator=g, device="cuda") * 2).to(dt)
    lse = torch.empty((len(lengths), Hkv * G), device="cuda")
    out = la.attend_decode(q, kc, vc, pages, ints(lengths), lse=lse, k_scale=ks, v_scale=vs)
    for b, (k, v) in enumerate(seqs):
        seen = torch.ones((1, lengths[b]), dtype=torch.bool, device="cuda")
        assert_attention(out[b:b + 1], lse[b:b + 1], q[b:b + 1], k, v, seen, D ** -0.5)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("new,ahead,Hkv,G,D,page,width,causal,order", [
    ([1], [0], 1, 1, 16, 8, None, True, "rows"), ([5, 0, 33], [3, 9, 0], 2, 3, 64, 8, None, True, "rows"), ([130, 17], [0, 100], 2, 4, 128, 16, None, True, "rows"),
    ([64, 65], [63, 1], 1, 5, 96, 24, None, True, "heads"), ([40], [30], 2, 2, 256, 16, None, True, "rows"), ([33, 90], [31, 200], 1, 8, 192, 32, None, False, "rows"),
    ([100], [900], 1, 8, 128, 16, None, True, "rows"), ([300, 20], [500, 1300], 2, 4, 128, 16, 200, True, "rows"), ([50], [700], 2, 1, 80, 16, None, False, "heads"),
    ([70, 3], [600, 0], 1, 4, 256, 16, 80, True, "rows")])
def test_prompt(la, code, dt, new, ahead, Hkv, G, D, page, width, causal, order):
    g, dt = gen(sum(new) + D), DT[dt]
    lengths = [n + a for n, a in zip(new, ahead)]
    kc, vc, ks, vs, pages, seqs = paged8(g, lengths, page, Hkv, D, dt, CODES[code], width=width, order=order)
    pad = 2
    starts = [pad + sum(new[:i]) for i in range(len(new) + 1)]
    q = (torch.randn((starts[-1] + pad, Hkv * G, D), generator=g, device="cuda") * 2).to(dt)
    out = torch.full_like(q, 7.0)
    lse = torch.full(q.shape[:2], 7.0, device="cuda")
    for with_lse in (True, False):
        la.attend_prompt_paged(q, kc, vc, pages, ints(lengths), ints(starts), causal=causal, out=out, lse=lse if with_lse else None, k_scale=ks, v_scale=vs)
        for b, (k, v) in enumerate(seqs):
            s = slice(starts[b], starts[b + 1])
            assert_attention(out[s], lse[s] if with_lse else None, q[s], k, v, visible(new[b], lengths[b], causal, "cuda"), D ** -0.5)
        for t in (out, lse):
            assert bool((t[:pad] == 7).all()) and bool((t[starts[-1]:] == 7).all())


@pytest.mark.parametrize("code", ["16", *CODES])
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("shared,lengths,Hkv,G,D,page,width", [
    (1, [9, 8, 20], 1, 1, 16, 8, None), (2, [40, 0, 33, 32, 31, 5], 2, 4, 64, 16, None), (8, [130, 128, 300, 129], 2, 3, 128, 16, None), (5, [80] * 9, 1, 16, 96, 16, 5),
    (40, [700, 641, 640, 1200, 0, 12], 2, 8, 128, 16, 100), (70, [1200, 1121, 4], 1, 5, 256, 16, None), (130, [2100] * 40, 1, 4, 128, 16, None), (4, [70], 2, 2, 192, 16, None),
    # So many numbers that the prefix goes by itself: rows of several tiles, of one, splits that end inside a chunk, lengths inside the prefix.
    (32, [4097, 4096, 0, 4095, 700, 5000] * 10, 2, 3, 128, 128, None), (257, [4112 + 7 * i for i in range(130)], 1, 5, 64, 16, None),
    (64, [4096, 4100, 30, 4400] * 10, 1, 2, 256, 64, 80), (256, [4096] * 80, 1, 1, 96, 16, None), (130, [2080 + i % 40 for i in range(150)], 1, 18, 128, 16, None)])
def test_decode_over_a_shared_prefix(la, code, dt, shared, lengths, Hkv, G, D, page, width):
    g, dt = gen(sum(lengths) + D), DT[dt]
    c = torch.int8 if code == "16" else CODES[code]
    kc, vc, ks, vs, pages, seqs = paged8(g, lengths, page, Hkv, D, dt, c, width=width, shared=shared)
    prefix = pages[0, :shared].clone()
    pages[1:, :shared] = -5  # not looked at
    scales = dict(k_scale=ks, v_scale=vs)
    if code == "16":  # the same numbers, rounded; what is unused is NaN
        kc, vc = ((x.float() * s.transpose(1, 2)[..., None]).to(dt) for x, s in ((kc, ks), (vc, vs)))
        seqs = [tuple(x.to(dt) for x in kv) for kv in seqs]
        scales = {}
    B, H = len(lengths), Hkv * G
    q = (torch.randn((B, H, D), generator=g, device="cuda") * 2).to(dt)
    lse = torch.empty((B, H), device="cuda")
    out = la.attend_decode_shared(q, kc, vc, prefix, pages, ints(lengths), lse=lse, **scales)
    for b, (k, v) in enumerate(seqs):
        seen = torch.ones((1, lengths[b]), dtype=torch.bool, device="cuda")
        assert_attention(out[b:b + 1], lse[b:b + 1], q[b:b + 1], k, v, seen, D ** -0.5)
    again = la.attend_decode_shared(q, kc, vc, prefix, pages, ints(lengths), **scales)
    assert torch.equal(again, out)  # and without the log-sum-exp


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("kind", ["zero values", "scale 0", "tiny values", "one key", "far scales"])
def test_rows_whose_scales_differ_widely(la, code, dt, kind):
    """Zero rows weigh in the sum, tiny ones keep what the type holds, and a row that one key makes is that key's value, rounded once."""
    g, dt, D, m = gen(21), DT[dt], 64, 200
    kc, vc, ks, vs, pages, seqs = paged8(g, [m], 16, 1, D, dt, CODES[code])
    k, v = seqs[0]
    rows, at = pages[0].long()[torch.arange(m, device="cuda") // 16], torch.arange(m, device="cuda") % 16
    by = torch.ones(m, device="cuda", dtype=torch.float64)
    if kind == "zero values":
        by[::2] = 0.0
    elif kind == "scale 0":
        by[1::3] = 0.0
    elif kind == "tiny values":
        by *= 2.0 ** -22 if dt == torch.float16 else 2.0 ** -110
    elif kind == "far scales":
        by = torch.exp2(torch.randint(-20, 7, (m,), generator=g, device="cuda").double())
    if kind == "zero values":  # as kv_append stores them
        codes, scale = quantise(torch.zeros((m, 1, D), device="cuda"), CODES[code])
        keep = by > 0
        put(vc, (rows[~keep], at[~keep]), codes[~keep])
        vs[rows[~keep], :, at[~keep]] = scale[~keep]
    else:
        vs[rows, :, at] = (vs[rows, :, at].double() * by[:, None]).float()
    v = v * by[:, None, None]
    q = torch.randn((3, 2, D), generator=g, device="cuda").to(dt)
    q = q * 30 if kind == "one key" else q
    scales = dict(k_scale=ks, v_scale=vs)
    lse = torch.empty((3, 2), device="cuda")
    out = la.attend_prompt_paged(q, kc, vc, pages, ints([m]), ints([0, 3]), lse=lse, **scales)
    assert_attention(out, lse, q, k, v, visible(3, m, True, "cuda"), D ** -0.5)
    out = la.attend_decode(q[2:], kc, vc, pages, ints([m]), lse=lse[2:], **scales)
    assert_attention(out, lse[2:], q[2:], k, v, visible(1, m, False, "cuda"), D ** -0.5)
    out = la.attend_decode_shared(q[2:], kc, vc, pages[0, :5], pages, ints([m]), lse=lse[2:], **scales)
    assert_attention(out, lse[2:], q[2:], k, v, visible(1, m, False, "cuda"), D ** -0.5)
    if kind == "one key":  # the nearest the type has, but for the others' share
        p = torch.softmax((q[2].double() @ k[:, 0].T) * D ** -0.5, -1)
        sure = p.amax(-1) > 1 - 2.0 ** -14
        got, want = out[0], p @ v[:, 0]
        u = torch.finfo(dt).eps / 2
        assert bool(((got.double() - want).abs() <= want.abs() * u * 1.02 + v.abs().amax() * 2.0 ** -13)[sure].all())


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("most", [1.75, 2.0, 3.96875, 1.0078125])
def test_codes_are_nearest_ones(la, code, dt, most):
    """x top / m in 64 bits is no further from its code than half a step and three roundings of fp32 (reciprocal, two products)."""
    code, dt = CODES[code], DT[dt]
    x = (torch.arange(8 * 256, device="cuda").view(8, 1, 256) / 2048 * most).to(dt)
    x[:, :, 0] = most
    kc, ks = empty_cache(1, 8, 1, 256, code)
    vc, vs = empty_cache(1, 8, 1, 256, code)
    la.kv_append(x, -x, kc, vc, ints([[0]]), ints(range(8)), seqs=ints([0] * 8), k_scale=ks, v_scale=vs)
    m = x.double().abs().amax(-1, keepdim=True)
    y = (x.double() * (127 if code == torch.int8 else 448) / m).squeeze(1)
    step = torch.ones_like(y) if code == torch.int8 else torch.exp2(y.clamp(min=2.0 ** -6).log2().floor() - 3)
    for c, sign in ((kc, 1), (vc, -1)):
        assert bool(((sign * take(c, 0).float().double().squeeze(1) - y).abs() <= step / 2 + y * 3 * 2.0 ** -24).all())
