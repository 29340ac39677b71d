"""What a served decoder layer needs beyond 16-bit attention: the calls its speed is judged by.

Four groups around the paged key-value cache and the residual stream:

  append  kv_append into an 8-bit cache (a scale a token and head), the queries
          rotated with it, and kv_read of what it holds then
  decode  attend_decode over such a cache
  prompt  attend_prompt_paged over such a cache
  shared  attend_decode_shared: one new token for each of a batch that has its
          first positions in common, over 8-bit and 16-bit caches
  norm    residual_norm: x' = x + scale gate post(y), n = pre(x')

An 8-bit row of D numbers x has the scale s = max|x| / top (top: 127 for int8,
448 for float8_e4m3fn) and the codes round(x (top / max|x|)).  `plain_*` compute
the operators with elementary torch operations in 32 bits, `exact_*` in 64.
With `own` set, `run` calls the library.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
CODES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "fp8": 448.0}
LEAST = 2.0 ** -100  # a row's largest magnitude counts as no less
WIDE = {"Hq": 64, "Hkv": 8, "D": 128}
USUAL = {"Hq": 32, "Hkv": 8, "D": 128}


def listed():
    return [
        # One user's next token: latency.
        dict(name="append_1", kind="append", T=1, B=1, far=1000, rot=128, inter=False, page=16, dtype="bf16", cache="int8", mix=1,
             **USUAL),
        # A decode batch; half of each head rotated, neighbours as pairs.
        dict(name="append_200", kind="append", T=200, B=200, far=2000, rot=32, inter=True, page=64, dtype="f16", cache="fp8", mix=2,
             Hq=28, Hkv=4, D=64),
        # Prompts of several users at once, one of them far into a long context.
        dict(name="append_8190", kind="append", T=8190, B=5, far=60000, rot=128, inter=False, page=32, dtype="bf16", cache="int8",
             mix=3, **WIDE),
        # One user, a short conversation: latency.
        dict(name="decode_1", kind="decode", B=1, L=301, spread=1, empty=0, page=16, lse=False, dtype="bf16", cache="int8", mix=4,
             **USUAL),
        # A padded batch of conversations of very different lengths.
        dict(name="decode_35_ragged", kind="decode", B=35, L=16000, spread=1000, empty=3, page=16, lse=True, dtype="bf16",
             cache="fp8", mix=5, **USUAL),
        # A server's whole cache.
        dict(name="decode_64_full", kind="decode", B=64, L=20000, spread=2, empty=0, page=128, lse=False, dtype="f16", cache="int8",
             mix=6, **WIDE),
        # The next 500 or so tokens of long prompts, in front of them what is cached.
        dict(name="prompt_4_chunks", kind="prompt", B=4, L=517, spread=2, ahead=9000, page=32, causal=True, lse=False, dtype="bf16",
             cache="fp8", mix=7, **USUAL),
        # Long prompts behind longer ones.
        dict(name="prompt_2_long", kind="prompt", B=2, L=4099, spread=1, ahead=8000, page=64, causal=True, lse=True, dtype="f16",
             cache="int8", mix=8, **USUAL),
        # A few users of one assistant: its instructions are the same for all.
        dict(name="shared_5", kind="shared", B=5, P=4096, L=700, spread=20, empty=1, page=16, lse=False, dtype="bf16", cache="16",
             mix=9, **USUAL),
        # Many questions about one long document.
        dict(name="shared_64", kind="shared", B=64, P=16000, L=2000, spread=50, empty=0, page=64, lse=True, dtype="bf16",
             cache="int8", mix=10, **WIDE),
        # Between two blocks of a step for one user: latency.
        dict(name="norm_1", kind="norm", T=1, d=4096, x="f32", y="bf16", n="bf16", post="rms", pre="rms", gate="row", by=0.5),
        # The same in a prefill batch, gates by token.
        dict(name="norm_8190", kind="norm", T=8190, d=7168, x="f32", y="f32", n="bf16", post="rms", pre="layer", gate="all", by=1.0),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(("append", "decode", "decode", "prompt", "shared", "shared", "norm"))
    if kind == "norm":
        d = rng.choice((_log(rng, 64, 16384), 8 * _log(rng, 8, 2048), 128 * _log(rng, 1, 128)))
        return dict(kind=kind, T=_log(rng, 1, min(16384, (1 << 25) // d)), d=d, x=rng.choice(("f32", "f32", "bf16")),
                    y=rng.choice(("none", "f32", "bf16", "f16")), n=rng.choice(("bf16", "f16", "f32")),
                    post=rng.choice(("none", "rms", "layer")), pre=rng.choice(("rms", "rms", "layer")),
                    gate=rng.choice(("none", "row", "all")), by=rng.choice((1.0, 0.5, 0.22)))
    D = rng.choice((64, 64, 80, 96, 128, 128, 128, 256))
    Hkv = rng.choice((1, 2, 4, 8, 8))
    G = rng.choice((1, 2, 3, 4, 5, 7, 8, 16))
    c = dict(kind=kind, Hq=Hkv * G, Hkv=Hkv, D=D, page=rng.choice((16, 16, 32, 48, 64, 128)),
             dtype=rng.choice(("bf16", "bf16", "f16")), cache=rng.choice(("int8", "fp8")), mix=rng.randrange(1 << 20))
    row = Hkv * D * 4  # bytes of a token's key and value in 16 bits
    if kind == "append":
        one = rng.random() < 0.5  # a token a sequence, or prompts
        B = _log(rng, 1, 256) if one else _log(rng, 1, 16)
        T = B if one else max(B, _log(rng, 16, 8192))
        far = _log(rng, 64, max(64, min(100000, (1 << 30) // (row * B))))
        T = min(T, B * (far // 2))
        return dict(c, T=T, B=B, far=far, rot=rng.choice((D, D, D // 2)), inter=rng.random() < 0.3)
    if kind == "decode":
        B = _log(rng, 1, 200)
        L = _log(rng, 1, max(1, min(120000, (3 << 30) // (row * B), (12 << 30) // (c["Hq"] * 4 * B))))
        return dict(c, B=B, L=L, spread=rng.choice((1, 2, 20, 400)), empty=rng.randrange(3) if B > 8 else 0, lse=rng.random() < 0.5)
    if kind == "shared":
        B = _log(rng, 2, 200)
        P = c["page"] * max(1, _log(rng, 256, max(256, min(60000, (8 << 30) // (c["Hq"] * 4 * B)))) // c["page"])
        L = _log(rng, 1, max(1, min(4000, (2 << 30) // (row * B))))
        return dict(c, B=B, P=P, L=L, spread=rng.choice((1, 2, 20, 400)), empty=rng.randrange(3) if B > 8 else 0, lse=rng.random() < 0.5,
                    cache=rng.choice(("16", "16", "int8", "fp8")))
    B = _log(rng, 1, 24)
    # Scores that the plain form holds: B Hq L (L + ahead) values, at most 2^30.
    L = _log(rng, 1, max(1, min(4000, int(math.sqrt((1 << 29) / (B * c["Hq"]))))))
    ahead = _log(rng, 1, max(1, min(8000, (1 << 29) // (B * c["Hq"] * L))))
    return dict(c, B=B, L=L, spread=rng.choice((1, 2, 20)), ahead=ahead, causal=rng.random() < 0.8, lse=rng.random() < 0.5)


# ---- lengths, from the case alone ----------------------------------------------
def _spread(rng, n, top, spread):
    """n lengths, the longest `top`, the others down to top / spread."""
    low = max(1, top // spread)
    return [top] + [_log(rng, low, top) if low < top else top for _ in range(n - 1)]


def _token_lengths(c):
    """Positions of each sequence: all of them, or behind the shared ones."""
    rng = random.Random(c["mix"])
    got = _spread(rng, c["B"] - c["empty"], c["L"], c["spread"]) + [0] * c["empty"]
    rng.shuffle(got)
    return got


def _prompt_lengths(c):
    """(new tokens, keys) of each sequence."""
    rng = random.Random(c["mix"])
    new = _spread(rng, c["B"], c["L"], c["spread"])
    return new, [n + _log(rng, 1, c["ahead"]) for n in new]


def _append_tokens(c):
    """(tokens, first position) of each sequence."""
    rng = random.Random(c["mix"])
    cuts = sorted(rng.sample(range(1, c["T"]), c["B"] - 1)) if c["B"] < c["T"] else list(range(1, c["B"]))
    new = [b - a for a, b in zip([0] + cuts, cuts + [c["T"]])]
    new = new if max(new) <= c["far"] else [c["T"] // c["B"] + (i < c["T"] % c["B"]) for i in range(c["B"])]
    return new, [rng.randrange(c["far"] - n + 1) for n in new]


# ---- inputs --------------------------------------------------------------------
def _pages(gen, lengths, page, width):
    """Page table [B, width] of pages in no order, -1 behind a sequence's last; the pages left over."""
    need = torch.tensor([-(-n // page) for n in lengths], device="cuda")
    total = int(need.sum()) + 7
    order = torch.randperm(total, generator=gen, device="cuda").int()
    at = torch.arange(width, device="cuda")[None, :]
    first = (need.cumsum(0) - need)[:, None]
    table = torch.where(at < need[:, None], order[(first + at).clamp(max=total - 1)], torch.full((), -1, dtype=torch.int32, device="cuda"))
    return table.contiguous(), total


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _starts(lengths):
    return _ints([sum(lengths[:i]) for i in range(len(lengths) + 1)])


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, by=1.0, dt=None):
        return torch.randn(shape, generator=gen, device="cuda", dtype=DTYPES[dt or c["dtype"]]).mul_(by)

    s = dict(c)
    if c["kind"] == "norm":
        T, d = c["T"], c["d"]
        s.update(x=normal(T, d, by=3.0, dt=c["x"]), y=None if c["y"] == "none" else normal(T, d, by=0.7, dt=c["y"]),
                 gate=None if c["gate"] == "none" else normal(*((d,) if c["gate"] == "row" else (T, d)), by=0.3, dt="f32"))
        for n in ("post", "pre"):
            s[n + "_w"] = None if c[n] == "none" else normal(d, by=0.2, dt="f32").add_(1.0)
            s[n + "_b"] = normal(d, by=0.1, dt="f32") if c[n] == "layer" else None
        return s
    Hq, Hkv, D, page = c["Hq"], c["Hkv"], c["D"], c["page"]

    def cache(n):
        """Keys with channels of very different size, values; rows of either of different size."""
        for name in ("k", "v"):
            x = normal(n, page, Hkv, D)
            x *= torch.exp2(torch.randn((n, page, Hkv, 1), generator=gen, device="cuda")).to(x.dtype)
            if name == "k":
                x *= torch.exp2(0.8 * torch.randn((1, 1, Hkv, D), generator=gen, device="cuda") - 0.8).to(x.dtype)
            if c["cache"] == "16":
                s[name + "_cache"], s[name + "_scale"] = x, None
            else:
                codes, scale = plain_quantise(x, c["cache"])
                s[name + "_cache"], s[name + "_scale"] = codes, scale.transpose(1, 2).contiguous()

    if c["kind"] == "append":
        new, first = _append_tokens(c)
        pages, n = _pages(gen, [c["far"]] * c["B"], page, -(-c["far"] // page))
        positions = [p for a, k in zip(first, new) for p in range(a, a + k)]
        cache(n)
        # The projection's fused output: q, k and v are views of it.
        qkv = normal(c["T"], Hq + 2 * Hkv, D)
        angle = torch.arange(c["far"], device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (
            -torch.arange(0, c["rot"], 2, device="cuda", dtype=torch.float64) / c["rot"])
        s.update(q=qkv[:, :Hq], k=qkv[:, Hq:Hq + Hkv], v=qkv[:, Hq + Hkv:], pages=pages, positions=_ints(positions),
                 seqs=_ints([b for b, k in enumerate(new) for _ in range(k)]),
                 rope=torch.stack((angle.cos(), angle.sin()), 1).float().contiguous())
        return s
    if c["kind"] == "prompt":
        new, lengths = _prompt_lengths(c)
        s.update(q=normal(sum(new), Hq, D, by=2.0), starts=_starts(new), new=_ints(new))
    else:
        lengths = _token_lengths(c)
        s.update(q=normal(c["B"], Hq, D, by=2.0))
    if c["kind"] == "shared":
        # The prefix's pages are the first that a table of one more sequence names.
        prefix = c["P"] // page
        pages, n = _pages(gen, [c["P"]] + lengths, page, max(prefix, -(-max(lengths) // page)))
        s.update(prefix=pages[0, :prefix].contiguous(),
                 pages=torch.cat((pages[0, :prefix].expand(c["B"], prefix), pages[1:, :-(-max(lengths) // page)]), 1).contiguous())
        # An empty slot has no positions at all.
        lengths = [c["P"] + m if m else 0 for m in lengths]
    else:
        pages, n = _pages(gen, lengths, page, -(-max(lengths) // page))
        s.update(pages=pages)
    cache(n)
    rows = s["q"].shape[0]
    s.update(lengths=_ints(lengths), lse_out=torch.empty((rows, Hq), dtype=torch.float32, device="cuda") if c["lse"] else None)
    return s


# ---- plain forms ---------------------------------------------------------------
def plain_quantise(x, kind):
    """Codes, and a scale for each row of the last dimension."""
    x = x.float()
    most = x.abs().amax(-1).clamp(min=LEAST)
    y = x * (TOP[kind] / most)[..., None]
    return (y.round() if kind == "int8" else y).to(CODES[kind]), most / TOP[kind]


def _taken(cache, index):
    """cache[index]; codes of 8-bit floating point travel as bytes."""
    return cache.view(torch.uint8)[index].view(cache.dtype) if cache.dtype == torch.float8_e4m3fn else cache[index]


def _rotated(x, cos, sin, rot, inter):
    """x [T, H, D] in 32 bits, its first `rot` dimensions rotated by cos, sin [T, rot / 2]."""
    x = x.float()
    cos, sin = cos[:, None, :], sin[:, None, :]
    if inter:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def _stored(x, s, cache, scale, page, row):
    codes, sc = plain_quantise(x, s["cache"])
    s[cache].view(torch.uint8)[page, row] = codes.view(torch.uint8)
    s[scale][page, :, row] = sc
    return (_taken(s[cache], (page, row)).float() * s[scale][page, :, row][..., None]).to(s["q"].dtype)


def plain_append(s):
    at = s["positions"].long()
    page, row = s["pages"][s["seqs"].long(), at // s["page"]].long(), at % s["page"]
    cos, sin = s["rope"][at].unbind(1)
    k = _stored(_rotated(s["k"], cos, sin, s["rot"], s["inter"]), s, "k_cache", "k_scale", page, row)
    v = _stored(s["v"], s, "v_cache", "v_scale", page, row)
    q = _rotated(s["q"], cos, sin, s["rot"], s["inter"]).to(s["q"].dtype)
    return {"q": q, "k": k, "v": v, "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _cached(s, name, pages, m):
    """The first m rows of each sequence, [B, Hkv, m, D] in 32 bits."""
    B, n = pages.shape
    used = pages.clamp(min=0).long()
    x = _taken(s[name + "_cache"], used).float()
    if s[name + "_scale"] is not None:
        x *= s[name + "_scale"][used].transpose(2, 3)[..., None]
    return x.view(B, n * s["page"], s["Hkv"], s["D"])[:, :m].transpose(1, 2).contiguous()


def _scores(q, k):
    """q [B, Hq, n, D] over k [B, Hkv, m, D] -> [B, Hkv, G, n, m]."""
    B, Hq, n, D = q.shape
    Hkv, m = k.shape[1], k.shape[2]
    return torch.matmul(q.reshape(B, Hkv, Hq // Hkv * n, D), k.transpose(2, 3)).view(B, Hkv, Hq // Hkv, n, m).mul_(D ** -0.5)


def _softmax(x):
    """exp(x - top) in the place of x, its sum, the log-sum-exp; 0 and -inf where nothing is seen."""
    top = x.amax(-1, keepdim=True).nan_to_num_(neginf=0.0)
    x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    return torch.where(total > 0, total, 1.0), top + total.log()


def _attend(q, k, v, seen):
    B, Hq, n, D = q.shape
    x = _scores(q, k).masked_fill_(~seen[:, None, None], -math.inf)
    total, lse = _softmax(x)
    out = torch.matmul(x.flatten(2, 3), v).view(B, -1, Hq // k.shape[1], n, D) / total
    return out.reshape(B, Hq, n, D), lse.reshape(B, Hq, n)


def plain_decode(s):
    seen = torch.arange(s["L"], device="cuda")[None, None, :] < s["lengths"][:, None, None]
    out, lse = _attend(s["q"].float()[:, :, None, :], _cached(s, "k", s["pages"], s["L"]), _cached(s, "v", s["pages"], s["L"]), seen)
    return out[:, :, 0].to(s["q"].dtype), lse[:, :, 0]


def plain_shared(s):
    """The prefix's keys and values once, for the rows of all sequences; one softmax over both."""
    B, Hkv, G, D, P = s["B"], s["Hkv"], s["Hq"] // s["Hkv"], s["D"], s["P"]
    q = s["q"].float()
    pk, pv = (_cached(s, name, s["prefix"][None], P)[0] for name in ("k", "v"))
    own_pages = s["pages"][:, P // s["page"]:]
    m = min(s["L"], own_pages.shape[1] * s["page"])
    ok, ov = _cached(s, "k", own_pages, m), _cached(s, "v", own_pages, m)
    rows = q.view(B, Hkv, G, D).transpose(0, 1).reshape(Hkv, B * G, D)
    shared = torch.matmul(rows, pk.transpose(1, 2)).view(Hkv, B, G, P).transpose(0, 1).mul_(D ** -0.5)
    x = torch.cat((shared, _scores(q[:, :, None, :], ok)[:, :, :, 0]), -1)
    x.masked_fill_((torch.arange(P + m, device="cuda")[None, :] >= s["lengths"][:, None])[:, None, None], -math.inf)
    total, lse = _softmax(x)
    out = torch.matmul(x[..., :P].transpose(0, 1).reshape(Hkv, B * G, P), pv).view(Hkv, B, G, D).transpose(0, 1)
    out = (out + torch.matmul(x[..., P:], ov)) / total
    return out.reshape(B, Hkv * G, D).to(s["q"].dtype), lse.reshape(B, Hkv * G)


def plain_prompt(s):
    n, m, T = s["L"], s["pages"].shape[1] * s["page"], s["q"].shape[0]
    at = (s["starts"][:-1, None] + torch.arange(n, device="cuda")[None, :]).clamp(max=T - 1)
    q = s["q"][at.long()].transpose(1, 2).float().contiguous()
    i, j = torch.arange(n, device="cuda")[None, :, None], torch.arange(m, device="cuda")[None, None, :]
    seen = j < s["lengths"][:, None, None]
    seen = seen & (j <= i + (s["lengths"] - s["new"])[:, None, None]) if s["causal"] else seen.expand(-1, n, -1)
    out, lse = _attend(q, _cached(s, "k", s["pages"], m), _cached(s, "v", s["pages"], m), seen)
    row = torch.arange(T, device="cuda")
    b = torch.searchsorted(s["starts"][1:].contiguous(), row.int(), right=True)
    at = row - s["starts"][b]
    return out[b, :, at].to(s["q"].dtype), lse[b, :, at]


def _normed(x, kind, w, b, eps=1e-6):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w
    return x if b is None else x + b


def plain_norm(s):
    x = s["x"].float()
    if s["y"] is not None:
        y = s["y"].float()
        y = y if s["post"] == "none" else _normed(y, s["post"], s["post_w"], s["post_b"])
        x = x + s["by"] * (y if s["gate"] is None else y * s["gate"])
    return {"x": x.to(s["x"].dtype), "n": _normed(x, s["pre"], s["pre_w"], s["pre_b"]).to(DTYPES[s["n"]])}


# ---- one pass ------------------------------------------------------------------
def run(state):
    s = state
    if own:
        import latent_amd

        if s["kind"] == "norm":
            post, pre = (None if s[n] == "none" else latent_amd.Norm(s[n + "_w"], bias=s[n + "_b"], kind=s[n], eps=1e-6)
                         for n in ("post", "pre"))
            x, n = latent_amd.residual_norm(s["x"], s["y"], post=post if s["y"] is not None else None,
                                            gate=s["gate"] if s["y"] is not None else None, scale=s["by"], pre=pre, dtype=DTYPES[s["n"]])
            return {"x": x, "n": n}
        scales = dict(k_scale=s["k_scale"], v_scale=s["v_scale"])
        if s["kind"] == "append":
            q = latent_amd.kv_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["pages"], s["positions"], seqs=s["seqs"], q=s["q"],
                                     rope=s["rope"], interleaved=s["inter"], **scales)
            k, v = latent_amd.kv_read(s["k_cache"], s["v_cache"], s["pages"], s["positions"], seqs=s["seqs"], dtype=q.dtype, **scales)
            return {"q": q, "k": k, "v": v, "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
        if s["kind"] == "decode":
            out = latent_amd.attend_decode(s["q"], s["k_cache"], s["v_cache"], s["pages"], s["lengths"], lse=s["lse_out"], **scales)
        elif s["kind"] == "shared":
            out = latent_amd.attend_decode_shared(s["q"], s["k_cache"], s["v_cache"], s["prefix"], s["pages"], s["lengths"],
                                                  lse=s["lse_out"], **scales)
        else:
            out = latent_amd.attend_prompt_paged(s["q"], s["k_cache"], s["v_cache"], s["pages"], s["lengths"], s["starts"],
                                                 causal=s["causal"], lse=s["lse_out"], **scales)
        return {"out": out, "lse": s["lse_out"]} if s["lse"] else {"out": out}
    if s["kind"] in ("append", "norm"):
        return plain_append(s) if s["kind"] == "append" else plain_norm(s)
    out, lse = plain_decode(s) if s["kind"] == "decode" else plain_shared(s) if s["kind"] == "shared" else plain_prompt(s)
    return {"out": out, "lse": lse} if s["lse"] else {"out": out}


def work(case):
    c = case
    if c["kind"] == "norm":
        size = {"f32": 4, "bf16": 2, "f16": 2, "none": 0}
        some = c["y"] != "none"
        gate = 4 * some * {"none": 0, "row": 1, "all": c["T"]}[c["gate"]]
        return {"bytes": c["d"] * (c["T"] * (2 * size[c["x"]] + size[c["y"]] + size[c["n"]]) + gate + 8), "flops": 12 * c["T"] * c["d"]}
    Hq, Hkv, D = c["Hq"], c["Hkv"], c["D"]
    row = 4 * D if c["cache"] == "16" else 2 * D + 8  # key and value of a position and head
    if c["kind"] == "append":
        # q read and written, k and v read, stored, read and written; a row of the table a token.
        return {"bytes": c["T"] * (4 * Hq * D + 8 * Hkv * D + 2 * Hkv * row + 4 * c["rot"] + 8), "flops": c["T"] * (3 * (Hq + Hkv) * c["rot"] + 8 * Hkv * D)}
    if c["kind"] == "prompt":
        new, keys = _prompt_lengths(c)
        pairs = sum(a * b - (a * (a - 1) // 2 if c["causal"] else 0) for a, b in zip(new, keys))
        return {"bytes": Hkv * row * sum(keys) + 4 * Hq * D * sum(new), "flops": 4 * Hq * D * pairs}
    lengths = _token_lengths(c)
    shared = c["P"] if c["kind"] == "shared" else 0
    return {"bytes": Hkv * row * (shared + sum(lengths)) + 4 * Hq * D * c["B"],
            "flops": 4 * Hq * D * (sum(lengths) + shared * sum(n > 0 for n in lengths))}


# ---- 64 bits -------------------------------------------------------------------
def exact_append(c, s):
    at = s["positions"].long()
    cos, sin = s["rope"][at, 0].double(), s["rope"][at, 1].double()
    i = torch.arange(c["rot"] // 2, device="cuda")
    first, second = (2 * i, 2 * i + 1) if c["inter"] else (i, i + c["rot"] // 2)

    def turned(x):
        y = x.double()
        z = torch.complex(y[:, :, first], y[:, :, second]) * torch.complex(cos, sin)[:, None]
        y[:, :, first], y[:, :, second] = z.real, z.imag
        return y

    def nearest(y):
        """y to the nearest code's value: whole numbers, or steps of 2^-3 of a number's own power of two, 2^-9 at least."""
        step = torch.ones_like(y) if c["cache"] == "int8" else torch.exp2(y.abs().clamp(min=2.0 ** -6).log2().floor() - 3)
        return (y / step).round() * step

    got = {"q": turned(s["q"])}
    page = s["pages"].long()[s["seqs"].long(), at // c["page"]]
    for name, x in (("k", turned(s["k"])), ("v", s["v"].double())):
        scale = x.abs().amax(-1) / TOP[c["cache"]]
        got[name] = nearest(x / scale[..., None]) * scale[..., None]
        whole = s[name + "_scale"].double()
        whole.transpose(1, 2)[page, at % c["page"]] = scale
        got[name + "_scale"] = whole
    return got


def exact_norm(c, s):
    def normed(x, n):
        mean = x.mean(-1, keepdim=True) if c[n] == "layer" else torch.zeros_like(x[:, :1])
        x = (x - mean) / ((x - mean).pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * s[n + "_w"].double()
        return x + s[n + "_b"].double() if c[n] == "layer" else x

    x = s["x"].double()
    if s["y"] is not None:
        y = s["y"].double() if c["post"] == "none" else normed(s["y"].double(), "post")
        x = x + c["by"] * y * (1.0 if s["gate"] is None else s["gate"].double())
    return {"x": x, "n": normed(x, "pre")}


def _softmax64(q, k, v, seen):
    """q [h, n, D], k and v [m, D], seen [n, m] or None, in 64 bits."""
    x = q @ k.T * (1.0 / math.sqrt(q.shape[-1]))
    if seen is not None:
        x = torch.where(seen, x, -math.inf)
    lse = torch.logsumexp(x, -1)
    return torch.exp(x - lse[..., None]) @ v, lse


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] in ("append", "norm"):
        return exact_append(c, s) if c["kind"] == "append" else exact_norm(c, s)
    # Sequence by sequence, kv head by kv head, a block of query rows at a time.
    new, keys = _prompt_lengths(c) if c["kind"] == "prompt" else ([1] * c["B"], [int(n) for n in s["lengths"].tolist()])
    G = c["Hq"] // c["Hkv"]
    out = torch.zeros((sum(new), c["Hq"], c["D"]), dtype=torch.float64, device="cuda")
    lse = torch.full((sum(new), c["Hq"]), -math.inf, dtype=torch.float64, device="cuda")

    def values(name, pages, m, h):
        x = s[name + "_cache"][:, :, h]
        x = (x.view(torch.uint8)[pages].view(x.dtype) if c["cache"] == "fp8" else x[pages]).float().double()
        if c["cache"] != "16":
            x = x * s[name + "_scale"][pages][:, h].double()[..., None]
        return x.flatten(0, 1)[:m]

    at = 0
    for b, (n, m) in enumerate(zip(new, keys)):
        used = s["pages"][b, :-(-m // c["page"])].long()
        for h in range(c["Hkv"] if m else 0):
            kh, vh, heads = values("k", used, m, h), values("v", used, m, h), slice(h * G, (h + 1) * G)
            for r in range(0, n, 1024):
                e = min(n, r + 1024)
                seen = None
                if c.get("causal"):
                    seen = torch.arange(r, e, device="cuda")[:, None] + (m - n) >= torch.arange(m, device="cuda")[None, :]
                o, z = _softmax64(s["q"][at + r:at + e, heads].transpose(0, 1).double(), kh, vh, seen)
                out[at + r:at + e, heads], lse[at + r:at + e, heads] = o.transpose(0, 1), z.T
        at += n
    return {"out": out, "lse": lse} if c["lse"] else {"out": out}
