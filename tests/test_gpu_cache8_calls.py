"""Calls on 8-bit caches, shared prefixes and norms as a program makes them: refusals, streams, graphs, strides, NaN rows, large
offsets, workspaces, in-place counts, determinism."""

import math

import pytest
import torch

from tests._attention import assert_attention, visible
from tests._cache8 import CODES, bits, empty_cache, paged8, put, quantise, values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def la(gpu):
    return gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def calls(la, code=torch.int8, seed=0, lengths=(40, 300, 17), shared=1, Hkv=2, G=4, D=64, dt=torch.float16):
    """name -> f(**changes) on operands that fit."""
    g = gen(seed)
    kc, vc, ks, vs, pages, seqs = paged8(g, list(lengths), 16, Hkv, D, dt, code, shared=shared)
    B, H = len(lengths), Hkv * G
    q = torch.randn((B, H, D), generator=g, device="cuda").to(dt)
    kv = torch.randn((B, Hkv, D), generator=g, device="cuda").to(dt)
    n, T = ints(lengths), ints([0, 1, 2, 3][:B + 1])
    base = dict(k_cache=kc, v_cache=vc, pages=pages, k_scale=ks, v_scale=vs)
    return {
        "kv_append": lambda **c: la.kv_append(**{**base, **dict(k=kv, v=kv, positions=n - 1, q=q), **c}),
        "kv_read": lambda **c: la.kv_read(**{**base, **dict(positions=n - 1, dtype=dt), **c}),
        "attend_decode": lambda **c: la.attend_decode(**{**base, **dict(q=q, lengths=n), **c}),
        "attend_prompt_paged": lambda **c: la.attend_prompt_paged(**{**base, **dict(q=q, lengths=n, starts=T), **c}),
        "attend_decode_shared": lambda **c: la.attend_decode_shared(**{**base, **dict(q=q, lengths=n, prefix=pages[0, :shared]), **c}),
    }, base, seqs, q


NAMES = ["kv_append", "kv_read", "attend_decode", "attend_prompt_paged", "attend_decode_shared"]


@pytest.mark.parametrize("name", NAMES)
def test_refusals(la, name):
    f, base, _, q = calls(la)
    f = f[name]
    f()
    kc, ks = base["k_cache"], base["k_scale"]
    bad = [(dict(k_scale=None), TypeError), (dict(v_scale=None), TypeError), (dict(k_scale=ks[:, :1]), ValueError), (dict(k_scale=ks.half()), ValueError),
           (dict(v_scale=ks.cpu()), ValueError), (dict(v_scale=ks.transpose(1, 2).contiguous().transpose(1, 2)), ValueError), (dict(v_cache=kc.view(torch.float8_e4m3fn)), TypeError),
           (dict(v_cache=kc.half()), TypeError), (dict(k_cache=kc.view(torch.uint8), v_cache=kc.view(torch.uint8)), TypeError),
           (dict(k_cache=kc.half(), v_cache=kc.half()), ValueError),  # scales without codes
           (dict(k_cache=kc[:, :12], v_cache=kc[:, :12], k_scale=ks[..., :12], v_scale=ks[..., :12]), la.LatentError),
           (dict(k_scale=torch.zeros((*ks.shape[:2], 18), device="cuda")[..., :16]), la.LatentError)]  # heads 18 apart: no multiple of 4
    for change, error in bad:
        with pytest.raises(error):
            f(**change)
    if name != "kv_read":
        with pytest.raises(RuntimeError, match="backward"):
            f(k_scale=ks.clone().requires_grad_())
    if name == "attend_decode_shared":
        pages = base["pages"]
        for change, error in ((dict(prefix=pages[0, :1].long()), ValueError), (dict(prefix=pages[:, :1]), ValueError), (dict(prefix=None), TypeError),
                              (dict(prefix=pages[0, :1].cpu()), ValueError), (dict(prefix=ints([0] * (pages.shape[1] + 1))), ValueError)):
            with pytest.raises(error):
                f(**change)
    if name == "kv_read":
        for change, error in ((dict(dtype=None), TypeError), (dict(positions=ints([[0]])), ValueError), (dict(positions=ints([0] * 4)), ValueError),
                              (dict(seqs=ints([0])), ValueError)):
            with pytest.raises(error):
                f(**change)


def test_norm_refusals(la):
    x = torch.zeros((3, 64), device="cuda")
    w = torch.ones(64, device="cuda")
    ok = dict(x=x, y=x.clone(), post=la.Norm(w), gate=w, pre=la.Norm(w))
    la.residual_norm(**ok)
    for change, error in ((dict(x=x[0]), ValueError), (dict(y=x[:2]), ValueError), (dict(y=x.cpu()), ValueError), (dict(y=x.double()), TypeError), (dict(y=None), ValueError),
                          (dict(post=la.Norm(w[:8])), ValueError), (dict(pre=la.Norm(w.cpu())), ValueError), (dict(pre=la.Norm(w, bias=w.half())), TypeError),
                          (dict(gate=w[:8]), ValueError), (dict(gate=x[:2]), ValueError), (dict(gate=w.int()), TypeError), (dict(dtype=torch.int32), TypeError),
                          (dict(x_out=x.half()), ValueError), (dict(x_out=x[:1].expand(3, 64)), ValueError), (dict(n_out=x.half()), ValueError), (dict(n_out=x.t()), ValueError),
                          (dict(pre=None, n_out=x), ValueError), (dict(scale=math.nan), la.LatentError), (dict(scale=math.inf), la.LatentError),
                          (dict(x=torch.zeros((1, 40000), device="cuda"), y=None, post=None, gate=None, pre=la.Norm()), la.LatentError)):
        with pytest.raises(error):
            la.residual_norm(**{**ok, **change})
    for name in ("x", "y", "gate"):
        with pytest.raises(RuntimeError, match="backward"):
            la.residual_norm(**{**ok, name: ok[name].clone().requires_grad_()})
    with pytest.raises(RuntimeError, match="backward"):
        la.residual_norm(**{**ok, "pre": la.Norm(w.clone().requires_grad_())})
    with torch.no_grad():
        la.residual_norm(**{**ok, "x": x.clone().requires_grad_()})


@pytest.mark.parametrize("name", NAMES)
def test_another_stream_and_what_is_written_counts_as_changed(la, name):
    f, base, _, q = calls(la, seed=3)
    want = f[name]()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = f[name](stream=side)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got if isinstance(got, tuple) else (got,), want if isinstance(want, tuple) else (want,)):
        assert torch.equal(a, b)
    if name == "kv_append":
        tensors = [base[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale")]
        before = [t._version for t in tensors]
        f[name]()
        assert all(t._version > v for t, v in zip(tensors, before))


@pytest.mark.parametrize("code", CODES)
def test_captured_calls_replayed(la, code):
    """Each call in one graph, replayed with other inputs in the same places, against the eager calls; two graphs in turn."""
    f, base, _, q = calls(la, CODES[code], seed=4, lengths=(700, 45, 333), shared=2)
    x = torch.randn((3, 512), device="cuda")
    norm = la.Norm(torch.randn(512, device="cuda"))
    later = {n: f[n] for n in NAMES[1:]}
    more = lambda: la.residual_norm(x, x.clone(), post=norm, gate=norm.weight, pre=norm, dtype=torch.float16)  # noqa: E731
    f["kv_append"](), more(), [c() for c in later.values()]
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = [f["kv_append"](), *f["kv_read"](), f["attend_decode"](), f["attend_prompt_paged"](), f["attend_decode_shared"](), *more()]
        graphs.append((g, got))
    for i in range(4):
        q.copy_(torch.randn_like(q))
        x.copy_(torch.randn_like(x))
        want = [f["kv_append"](), *f["kv_read"](), f["attend_decode"](), f["attend_prompt_paged"](), f["attend_decode_shared"](), *more()]
        torch.cuda.synchronize()
        g, got = graphs[i % 2]
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), i


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_a_row_that_is_a_nan_reaches_those_who_see_it(la, code, dt):
    g = gen(6)
    lengths = [100, 100]
    kc, vc, ks, vs, pages, _ = paged8(g, lengths, 16, 1, 64, dt, CODES[code])
    q = torch.randn((40, 2, 64), generator=g, device="cuda").to(dt)
    starts = ints([0, 20, 40])  # query i of a sequence sees 81 + i keys
    scales = dict(k_scale=ks, v_scale=vs)
    for name, s in (("k", ks), ("v", vs)):
        was = s[pages[1, 5].long(), 0, 10].clone()  # position 90 of sequence 1
        s[pages[1, 5].long(), 0, 10] = math.nan
        out = la.attend_prompt_paged(q, kc, vc, pages, ints(lengths), starts, **scales)
        nan = torch.isnan(out).all(-1).all(-1)
        assert bool(nan[30:].all()) and bool(torch.isfinite(out[:30]).all()), name
        out = la.attend_decode(q[:2], kc, vc, pages, ints(lengths), **scales)
        assert bool(torch.isfinite(out[0]).all()) and bool(torch.isnan(out[1]).all())
        out = la.attend_decode(q[:2], kc, vc, pages, ints([90, 90]), **scales)
        assert bool(torch.isfinite(out).all())
        # Sequence 1's first six pages as a prefix: seen by who is long enough.
        tables = torch.cat((pages[1:, :6], pages[:1, :6]), 0)
        out = la.attend_decode_shared(q[:2], kc, vc, pages[1, :6], tables[[0, 0]], ints([96, 90]), **scales)
        assert bool(torch.isnan(out[0]).all()) and bool(torch.isfinite(out[1]).all())
        s[pages[1, 5].long(), 0, 10] = was


@pytest.mark.parametrize("name", ["attend_decode", "attend_prompt_paged", "attend_decode_shared"])
def test_pages_that_do_not_exist_are_masked(la, name):
    f, base, seqs, q = calls(la, seed=8, lengths=(64, 300, 17))
    pages = base["pages"].clone()
    pages[1, 2], pages[1, 18], pages[0, 3] = -1, 1 << 20, base["k_cache"].shape[0]
    lse = torch.empty(q.shape[:2], device="cuda")
    out = f[name](pages=pages, lse=lse)
    for b, (k, v) in enumerate(seqs):
        seen = torch.ones((1, len(k)), dtype=torch.bool, device="cuda")
        for p in {0: [3], 1: [2, 18], 2: []}[b]:
            seen[:, 16 * p:16 * p + 16] = False
        assert_attention(out[b:b + 1], lse[b:b + 1], q[b:b + 1], k, v, seen, 64 ** -0.5)
    if name == "attend_decode_shared":
        out = f[name](prefix=ints([-7]), lse=lse, lengths=ints([64, 300, 16]))
        for b, (k, v) in enumerate(seqs):
            n = 16 if b == 2 else len(k)
            seen = torch.arange(n, device="cuda")[None] >= 16
            assert_attention(out[b:b + 1], lse[b:b + 1], q[b:b + 1], k[:n], v[:n], seen, 64 ** -0.5)


def test_strided_operands(la):
    """Queries and outputs that are views, caches whose keys and values have other strides, scales of other strides."""
    f, base, seqs, q = calls(la, seed=9, D=128, G=2)
    want = {n: f[n]() for n in ("attend_decode", "attend_prompt_paged", "attend_decode_shared")}
    n, page, H, D = base["k_cache"].shape
    wide = torch.full((n, page, H, 2 * D + 16), 0x55, dtype=torch.int8, device="cuda")
    wide[..., 16:16 + D] = base["k_cache"]
    ks = torch.full((n, 2 * H + 1, page + 8), math.nan, device="cuda")
    ks[:, 1:1 + H, :page] = base["k_scale"]
    v = base["v_cache"].permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3)
    big = torch.zeros((3, 9, D), dtype=q.dtype, device="cuda")
    big[:, 3:3 + q.shape[1]] = q
    odd = torch.zeros(q.numel() + 1, dtype=q.dtype, device="cuda")[1:].view(q.shape)  # copied by the call
    odd.copy_(q)
    for name, w in want.items():
        for qq in (big[:, 3:3 + q.shape[1]], odd):
            out = torch.zeros_like(big)
            got = f[name](q=qq, k_cache=wide[..., 16:16 + D], v_cache=v, k_scale=ks[:, 1:1 + H, :page], out=out[:, 1:1 + q.shape[1]])
            assert torch.equal(got, w) and bool((out[:, 1 + q.shape[1]:] == 0).all()) and bool((out[:, 0] == 0).all())


def test_offsets_that_pass_32_bits(la):
    """A cache of 5 GB of codes: the last pages, written, read back and attended to."""
    page, Hkv, D = 128, 8, 128
    n = (5 << 30) // (page * Hkv * D)
    kc, vc = (torch.zeros((n, page, Hkv, D), dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = la.kv_scales(kc), la.kv_scales(vc)
    g = gen(11)
    m = 300
    pages, seqs, at = ints([[n - 1, 0, n - 2]]), ints([0] * m), ints(range(m))
    k, v = (torch.randn((m, Hkv, D), generator=g, device="cuda").bfloat16() for _ in range(2))
    s = dict(k_scale=ks, v_scale=vs)
    la.kv_append(k, v, kc, vc, pages, at, seqs=seqs, **s)
    kq, vq = (values(*quantise(x, torch.int8)) for x in (k, v))
    kr, vr = la.kv_read(kc, vc, pages, at, seqs=seqs, dtype=torch.bfloat16, **s)
    assert torch.equal(kr, kq.float().bfloat16()) and torch.equal(vr, vq.float().bfloat16())
    q = torch.randn((2, 16, D), generator=g, device="cuda").bfloat16()
    for out, r, seen in ((la.attend_decode(q[:1], kc, vc, pages, ints([m]), **s), q[:1], visible(1, m, True, "cuda")),
                         (la.attend_prompt_paged(q, kc, vc, pages, ints([m]), ints([0, 2]), **s), q, visible(2, m, True, "cuda")),
                         (la.attend_decode_shared(q[:1], kc, vc, pages[0, :2], pages, ints([m]), **s), q[:1], visible(1, m, True, "cuda"))):
        assert_attention(out, None, r, kq, vq, seen, D ** -0.5)


@pytest.mark.parametrize("name", ["attend_decode", "attend_prompt_paged", "attend_decode_shared"])
def test_equal_calls_give_equal_bits_and_lengths_are_cut(la, name):
    f, base, _, q = calls(la, seed=12, lengths=(2000, 100, 900), shared=3)
    want = f[name]()
    for _ in range(3):
        assert torch.equal(f[name](), want)
    room = base["pages"].shape[1] * 16
    assert torch.equal(f[name](lengths=ints([1 << 30, -5, 900]))[0], f[name](lengths=ints([room, 0, 900]))[0])
    out = f[name](lengths=ints([0, -1, -(1 << 31)]))
    assert bool((out == 0).all())


def test_a_workspace_of_ones_own(la):
    f, base, _, q = calls(la, seed=13, lengths=(700, 100, 900), shared=2)
    n, width = 3, base["pages"].shape[1]
    for name, size in (("attend_decode", la.attend_decode_workspace_size(n, 8, 2, 64, width, 16, codes=True)),
                       ("attend_decode_shared", la.attend_decode_shared_workspace_size(n, 8, 2, 64, width, 16, 2, codes=True))):
        guard = torch.full((size + 4096,), 0xA5, dtype=torch.uint8, device="cuda")
        got = f[name](workspace=guard[:size])
        assert torch.equal(got, f[name]()) and bool((guard[size:] == 0xA5).all())
        with pytest.raises(la.LatentError):
            f[name](workspace=guard[:size - 16])


def test_no_sequences_no_tokens(la):
    f, base, _, q = calls(la)
    none = dict(q=q[:0], pages=base["pages"][:0], lengths=ints([]))
    assert f["attend_decode"](**none).shape[0] == 0 and f["attend_decode_shared"](**none).shape[0] == 0
    assert f["attend_prompt_paged"](**none, starts=ints([0])).shape[0] == 0
    assert [t.shape[0] for t in f["kv_read"](positions=ints([]))] == [0, 0]
    want = f["attend_decode"]()
    assert torch.equal(f["attend_decode_shared"](prefix=ints([])), want)  # nothing shared: the plain call


@pytest.mark.parametrize("code", ["16", *CODES])
def test_a_prefix_by_itself_with_rows_and_pages_that_are_not_there(la, code):
    """A NaN among the prefix's rows reaches the sequences that are long enough, pages that do not exist are masked; in a graph too."""
    g, B, P, H, D = gen(14), 70, 2048, 2, 128
    lengths = [2100 if b % 2 else 1000 for b in range(B)]
    kc, vc, ks, vs, pages, seqs = paged8(g, lengths, 16, H, D, torch.bfloat16, torch.int8 if code == "16" else CODES[code], shared=P // 16)
    scales = dict(k_scale=ks, v_scale=vs)
    if code == "16":
        kc, vc = ((x.float() * s.transpose(1, 2)[..., None]).bfloat16() for x, s in ((kc, ks), (vc, vs)))
        seqs = [tuple(x.bfloat16() for x in kv) for kv in seqs]
        scales = {}
    q = torch.randn((B, 4, D), generator=g, device="cuda").bfloat16()
    prefix, n = pages[0, :P // 16].clone(), ints(lengths)
    assert la.attend_decode_shared_workspace_size(B, 4, H, D, pages.shape[1], 16, P // 16) > la.attend_decode_workspace_size(B, 4, H, D, pages.shape[1], 16)
    f = lambda: la.attend_decode_shared(q, kc, vc, prefix, pages, n, **scales)  # noqa: E731
    want = f()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = f()
    prefix[3], prefix[90] = -1, 1 << 30
    for _ in range(3):
        graph.replay()
        out = f()
        torch.cuda.synchronize()
        assert torch.equal(got, out) and not torch.equal(got, want)
    for b in (0, 1, 69):
        k, v = seqs[b]
        at = torch.arange(lengths[b], device="cuda")[None]
        seen = ~(((at >= 48) & (at < 64)) | ((at >= 1440) & (at < 1456)))
        assert_attention(out[b:b + 1], None, q[b:b + 1], k, v, seen, D ** -0.5)
    row = prefix[100].long()  # positions 1600 ..: past the short ones
    if code == "16":
        vc[row, 4, 1] = math.nan
    else:
        vs[row, 1, 4] = math.nan
    out = f()
    assert bool(torch.isfinite(out[::2]).all()) and bool(torch.isfinite(out[1::2, :2]).all()) and bool(torch.isnan(out[1::2, 2:]).all())
    assert bool((la.attend_decode_shared(q, kc, vc, prefix, pages, n * 0, **scales) == 0).all())


@pytest.mark.parametrize("code", CODES)
def test_more_sequences_than_lanes(la, code):
    """70 prompts, of none to 40 tokens behind up to 50 cached ones, one of them long; the same as single tokens."""
    g = gen(15)
    new = [(7 * i) % 41 for i in range(70)]
    new[33] = 300
    lengths = [n + (11 * i) % 51 for i, n in enumerate(new)]
    kc, vc, ks, vs, pages, seqs = paged8(g, lengths, 8, 2, 64, torch.float16, CODES[code])
    starts = [sum(new[:i]) for i in range(71)]
    q = torch.randn((starts[-1], 4, 64), generator=g, device="cuda").half()
    out = la.attend_prompt_paged(q, kc, vc, pages, ints(lengths), ints(starts), k_scale=ks, v_scale=vs)
    one = la.attend_decode(q[:70], kc, vc, pages, ints(lengths), k_scale=ks, v_scale=vs)
    for b, (k, v) in enumerate(seqs):
        s = slice(starts[b], starts[b + 1])
        assert_attention(out[s], None, q[s], k, v, visible(new[b], lengths[b], True, "cuda"), 64 ** -0.5)
        assert_attention(one[b:b + 1], None, q[b:b + 1], k, v, visible(1, lengths[b], True, "cuda"), 64 ** -0.5)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("G", [3, 20])
def test_tables_of_more_than_the_last_level_cache(la, code, G):
    """A page table wide enough that rows are read past that cache, of which most names nothing."""
    g, H, D = gen(16), 4, 128
    lengths = [1500, 0, 40, 333]
    kc, vc, ks, vs, pages, seqs = paged8(g, lengths, 16, H, D, torch.bfloat16, CODES[code], spare=20000)  # 20000 pages of 16 KB
    wide = torch.full((4, 20000), -1, dtype=torch.int32, device="cuda")
    wide[:, :pages.shape[1]] = pages
    q = torch.randn((4, H * G, D), generator=g, device="cuda").bfloat16()
    lse = torch.empty(q.shape[:2], device="cuda")
    for f in (lambda: la.attend_decode(q, kc, vc, wide, ints(lengths), lse=lse, k_scale=ks, v_scale=vs),
              lambda: la.attend_decode_shared(q, kc, vc, pages[0, :0], wide, ints(lengths), lse=lse, k_scale=ks, v_scale=vs),
              lambda: la.attend_prompt_paged(q, kc, vc, wide, ints(lengths), ints([0, 1, 2, 3, 4]), lse=lse, k_scale=ks, v_scale=vs)):
        out = f()
        for b, (k, v) in enumerate(seqs):
            assert_attention(out[b:b + 1], lse[b:b + 1], q[b:b + 1], k, v, visible(1, lengths[b], True, "cuda"), D ** -0.5)


def test_two_calls_at_once(la):
    """Calls on two streams, without workspaces: each has its own."""
    f, base, _, q = calls(la, seed=17, lengths=(3000, 100, 2900), shared=2)
    want = [f[n]() for n in ("attend_decode", "attend_prompt_paged", "attend_decode_shared")]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(5):
        got = [[f[n](stream=s) for n in ("attend_decode", "attend_prompt_paged", "attend_decode_shared")] for s in streams]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))


def test_norm_operands_of_other_strides(la):
    """Broadcast rows, rows apart, a stream that the call writes through; a row stride of zero is no output."""
    g = gen(18)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    row, y = r(1, 96), r(5, 96)
    x, n = la.residual_norm(row.expand(5, 96), y[:1].expand(5, 96), post=la.Norm(bias=r(96)), gate=r(5, 1).bfloat16(), pre=la.Norm(kind="layer"), dtype=torch.float16)
    for b in range(5):
        assert x.shape == (5, 96) and x.is_contiguous() and n.shape == (5, 96)
    one = la.residual_norm(row.repeat(5, 1), y[:1].repeat(5, 1), pre=la.Norm(kind="layer"), dtype=torch.float16)
    two = la.residual_norm(row.expand(5, 96), y[:1].expand(5, 96), pre=la.Norm(kind="layer"), dtype=torch.float16)
    assert all(torch.equal(a, b) for a, b in zip(one, two)) and bool((two[0] == two[0][0]).all())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    three = la.residual_norm(row.expand(5, 96), y[:1].expand(5, 96), pre=la.Norm(kind="layer"), dtype=torch.float16, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(three, two))
