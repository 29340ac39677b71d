"""The attention half of a decoder layer: the calls its speed is judged by.

Three operators around one paged key-value cache:

  append  kv_append: new keys (rotated by their positions) and values go to
          their rows of the cache's pages; the queries are rotated with them
  decode  attend_decode: one new token a sequence attends to the cache
  prompt  attend_prompt / attend_prompt_paged: whole prompts of different
          lengths, packed, causal; keys and values packed too, or from the
          cache (a chunk of a prompt behind the part that is cached)

`plain_*` compute them with elementary torch operations in 32 bits, `exact_*`
sequence by sequence in 64 bits.  With `own` set, `run` calls the library.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
WIDE = {"Hq": 64, "Hkv": 8, "D": 128}
USUAL = {"Hq": 32, "Hkv": 8, "D": 128}


def listed():
    return [
        # One user's next token: latency.
        dict(name="append_1", kind="append", T=1, B=1, far=1000, rot=128, inter=False, page=16, dtype="bf16", mix=1, **USUAL),
        # A decode batch; half of each head rotated, neighbours as pairs.
        dict(name="append_200", kind="append", T=200, B=200, far=2000, rot=32, inter=True, page=64, dtype="f16", mix=2,
             Hq=28, Hkv=4, D=64),
        # Prompts of several users at once, one of them far into a long context.
        dict(name="append_8190", kind="append", T=8190, B=5, far=60000, rot=128, inter=False, page=32, dtype="bf16", mix=3,
             **WIDE),
        # One user, a short conversation: latency.
        dict(name="decode_1", kind="decode", B=1, L=301, spread=1, empty=0, page=16, lse=False, dtype="bf16", mix=4, **USUAL),
        # One user at the end of a long document: all the chip for one sequence.
        dict(name="decode_1_long", kind="decode", B=1, L=131071, spread=1, empty=0, page=64, lse=True, dtype="bf16", mix=5,
             **WIDE),
        # A padded batch of conversations of very different lengths.
        dict(name="decode_35_ragged", kind="decode", B=35, L=16000, spread=1000, empty=3, page=16, lse=False, dtype="bf16",
             mix=6, **USUAL),
        # Small heads that share one key and value head.
        dict(name="decode_96_shared", kind="decode", B=96, L=2500, spread=4, empty=0, page=48, lse=True, dtype="f16", mix=7,
             Hq=20, Hkv=1, D=64),
        # A server's whole cache.
        dict(name="decode_64_full", kind="decode", B=64, L=20000, spread=2, empty=0, page=128, lse=False, dtype="bf16", mix=8,
             **WIDE),
        # One short prompt: latency.
        dict(name="prompt_77", kind="prompt", B=1, L=77, spread=1, ahead=0, paged=False, page=0, causal=True, lse=False,
             dtype="bf16", mix=9, **USUAL),
        # A prefill batch of prompts of different lengths.
        dict(name="prompt_14_packed", kind="prompt", B=14, L=2000, spread=20, ahead=0, paged=False, page=0, causal=True,
             lse=True, dtype="f16", mix=10, **USUAL),
        # The next 500 or so tokens of long prompts, in front of them what is cached.
        dict(name="prompt_4_chunks", kind="prompt", B=4, L=517, spread=2, ahead=9000, paged=True, page=32, causal=True,
             lse=False, dtype="bf16", mix=11, **USUAL),
        # One long prompt.
        dict(name="prompt_8192", kind="prompt", B=1, L=8192, spread=1, ahead=0, paged=False, page=0, causal=True, lse=False,
             dtype="bf16", mix=12, **WIDE),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(("append", "decode", "decode", "prompt", "prompt"))
    D = rng.choice((64, 64, 96, 128, 128, 128, 256))
    Hkv = rng.choice((1, 2, 4, 8, 8))
    G = rng.choice((1, 2, 3, 4, 5, 7, 8, 16))
    c = dict(kind=kind, Hq=Hkv * G, Hkv=Hkv, D=D, page=rng.choice((16, 16, 32, 48, 64, 128)),
             dtype=rng.choice(("bf16", "bf16", "f16")), mix=rng.randrange(1 << 20))
    row = Hkv * D * 4  # bytes of a token's key and value
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
        return dict(c, B=B, L=L, spread=rng.choice((1, 2, 20, 400)), empty=rng.randrange(3) if B > 8 else 0,
                    lse=rng.random() < 0.5)
    B = _log(rng, 1, 24)
    paged = rng.random() < 0.4
    # Scores that the plain form holds: B Hq L (L + ahead) values, at most 2^30.
    L = _log(rng, 1, max(1, min(8000, int(math.sqrt((1 << 29) / (B * c["Hq"]))))))
    ahead = _log(rng, 1, max(1, min(8000, (1 << 29) // (B * c["Hq"] * L)))) if paged else 0
    return dict(c, B=B, L=L, spread=rng.choice((1, 2, 20)), ahead=ahead, paged=paged, page=c["page"] if paged else 0,
                causal=rng.random() < 0.8, lse=rng.random() < 0.5)


# ---- lengths, from the case alone ----------------------------------------------
def _spread(rng, n, top, spread):
    """n lengths, the longest `top`, the others down to top / spread."""
    low = max(1, top // spread)
    return [top] + [_log(rng, low, top) if low < top else top for _ in range(n - 1)]


def _decode_lengths(c):
    rng = random.Random(c["mix"])
    got = _spread(rng, c["B"] - c["empty"], c["L"], c["spread"]) + [0] * c["empty"]
    rng.shuffle(got)
    return got


def _prompt_lengths(c):
    """(new tokens, keys) of each sequence."""
    rng = random.Random(c["mix"])
    new = _spread(rng, c["B"], c["L"], c["spread"])
    return new, [n + (_log(rng, 1, c["ahead"]) if c["ahead"] else 0) for n in new]


def _append_tokens(c):
    """(tokens, first position) of each sequence."""
    rng = random.Random(c["mix"])
    cuts = sorted(rng.sample(range(1, c["T"]), c["B"] - 1)) if c["B"] < c["T"] else list(range(1, c["B"]))
    new = [b - a for a, b in zip([0] + cuts, cuts + [c["T"]])]
    new = new if max(new) <= c["far"] else [c["T"] // c["B"] + (i < c["T"] % c["B"]) for i in range(c["B"])]
    return new, [rng.randrange(c["far"] - n + 1) for n in new]


# ---- inputs --------------------------------------------------------------------
def _pages(gen, lengths, page, width):
    """Page table [B, width] of pages in no order, -1 behind a sequence's last; the number of pages, a few of them unused."""
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
    dt = DTYPES[c["dtype"]]

    def normal(*shape, by=1.0):
        return torch.randn(shape, generator=gen, device="cuda", dtype=dt).mul_(by)

    s = dict(c)
    Hq, Hkv, D, page = c["Hq"], c["Hkv"], c["D"], c["page"]
    if c["kind"] == "append":
        new, first = _append_tokens(c)
        pages, n = _pages(gen, [c["far"]] * c["B"], page, -(-c["far"] // page))
        positions = [p for a, k in zip(first, new) for p in range(a, a + k)]
        # The projection's fused output: q, k and v are views of it.
        qkv = normal(c["T"], Hq + 2 * Hkv, D)
        angle = torch.arange(c["far"], device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (
            -torch.arange(0, c["rot"], 2, device="cuda", dtype=torch.float64) / c["rot"])
        s.update(q=qkv[:, :Hq], k=qkv[:, Hq:Hq + Hkv], v=qkv[:, Hq + Hkv:], pages=pages, positions=_ints(positions),
                 seqs=_ints([b for b, k in enumerate(new) for _ in range(k)]),
                 rope=torch.stack((angle.cos(), angle.sin()), 1).float().contiguous(),
                 k_cache=normal(n, page, Hkv, D), v_cache=normal(n, page, Hkv, D))
    elif c["kind"] == "decode":
        lengths = _decode_lengths(c)
        pages, n = _pages(gen, lengths, page, -(-max(lengths) // page))
        s.update(q=normal(c["B"], Hq, D, by=2.0), pages=pages, lengths=_ints(lengths), k_cache=normal(n, page, Hkv, D),
                 v_cache=normal(n, page, Hkv, D),
                 lse_out=torch.empty((c["B"], Hq), dtype=torch.float32, device="cuda") if c["lse"] else None)
    else:
        new, keys = _prompt_lengths(c)
        s.update(q=normal(sum(new), Hq, D, by=2.0), starts=_starts(new), new=_ints(new),
                 lse_out=torch.empty((sum(new), Hq), dtype=torch.float32, device="cuda") if c["lse"] else None)
        if c["paged"]:
            pages, n = _pages(gen, keys, page, -(-max(keys) // page))
            s.update(pages=pages, lengths=_ints(keys), k_cache=normal(n, page, Hkv, D), v_cache=normal(n, page, Hkv, D))
        else:
            s.update(k=normal(sum(new), Hkv, D), v=normal(sum(new), Hkv, D), lengths=_ints(new))
    return s


# ---- plain forms ---------------------------------------------------------------
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


def plain_append(s):
    at = s["positions"].long()
    page = s["pages"][s["seqs"].long(), at // s["page"]].long()
    cos, sin = s["rope"][at].unbind(1)
    dt = s["q"].dtype
    s["k_cache"][page, at % s["page"]] = _rotated(s["k"], cos, sin, s["rot"], s["inter"]).to(dt)
    s["v_cache"][page, at % s["page"]] = s["v"]
    return _rotated(s["q"], cos, sin, s["rot"], s["inter"]).to(dt)


def _attend(q, k, v, seen):
    """q [B, Hq, n, D], k and v [B, Hkv, m, D] in 32 bits, seen [B, n, m] -> out, log-sum-exp; 0 and -inf where nothing is seen."""
    B, Hq, n, D = q.shape
    Hkv, m = k.shape[1], k.shape[2]
    x = torch.matmul(q.reshape(B, Hkv, Hq // Hkv * n, D), k.transpose(2, 3)).view(B, Hkv, Hq // Hkv, n, m).mul_(D ** -0.5)
    x.masked_fill_(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True).nan_to_num_(neginf=0.0)
    x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    out = torch.matmul(x.view(B, Hkv, Hq // Hkv * n, m), v).view(B, Hkv, Hq // Hkv, n, D) / torch.where(total > 0, total, 1.0)
    return out.reshape(B, Hq, n, D), (top + total.log()).reshape(B, Hq, n)


def _cached(cache, pages, m):
    """The first m rows of each sequence, [B, Hkv, m, D] in 32 bits."""
    B, n = pages.shape
    rows = cache[pages.clamp(min=0).long()].view(B, n * cache.shape[1], cache.shape[2], cache.shape[3])
    return rows[:, :m].transpose(1, 2).float().contiguous()


def plain_decode(s):
    m = min(s["L"], s["pages"].shape[1] * s["page"])
    seen = torch.arange(m, device="cuda")[None, None, :] < s["lengths"][:, None, None]
    out, lse = _attend(s["q"].float()[:, :, None, :], _cached(s["k_cache"], s["pages"], m), _cached(s["v_cache"], s["pages"], m), seen)
    return out[:, :, 0].to(s["q"].dtype), lse[:, :, 0]


def _padded(x, starts, lengths, n):
    """Packed [T, H, D] as [B, H, n, D] in 32 bits."""
    at = (starts[:-1, None] + torch.arange(n, device="cuda")[None, :]).clamp(max=x.shape[0] - 1)
    return x[at.long()].transpose(1, 2).float().contiguous()


def plain_prompt(s):
    q = _padded(s["q"], s["starts"], s["new"], s["L"])
    if s["paged"]:
        m = s["pages"].shape[1] * s["page"]
        k, v = _cached(s["k_cache"], s["pages"], m), _cached(s["v_cache"], s["pages"], m)
    else:
        m = s["L"]
        k, v = _padded(s["k"], s["starts"], s["lengths"], m), _padded(s["v"], s["starts"], s["lengths"], m)
    i, j = torch.arange(s["L"], device="cuda")[None, :, None], torch.arange(m, device="cuda")[None, None, :]
    ahead = (s["lengths"] - s["new"])[:, None, None]
    seen = j < s["lengths"][:, None, None]
    seen = seen & (j <= i + ahead) if s["causal"] else seen.expand(-1, s["L"], -1)
    out, lse = _attend(q, k, v, seen)
    T = s["q"].shape[0]
    row = torch.arange(T, device="cuda")
    b = torch.searchsorted(s["starts"][1:].contiguous(), row.int(), right=True)
    at = row - s["starts"][b]
    return out[b, :, at].to(s["q"].dtype), lse[b, :, at]


# ---- one pass ------------------------------------------------------------------
def run(state):
    s = state
    if own:
        import latent_amd

        if s["kind"] == "append":
            q = latent_amd.kv_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["pages"], s["positions"], seqs=s["seqs"],
                                     q=s["q"], rope=s["rope"], interleaved=s["inter"])
            return {"q": q, "k": s["k_cache"], "v": s["v_cache"]}
        if s["kind"] == "decode":
            out = latent_amd.attend_decode(s["q"], s["k_cache"], s["v_cache"], s["pages"], s["lengths"], lse=s["lse_out"])
        elif s["paged"]:
            out = latent_amd.attend_prompt_paged(s["q"], s["k_cache"], s["v_cache"], s["pages"], s["lengths"], s["starts"],
                                                 causal=s["causal"], lse=s["lse_out"])
        else:
            out = latent_amd.attend_prompt(s["q"], s["k"], s["v"], s["starts"], causal=s["causal"], lse=s["lse_out"])
        return {"out": out, "lse": s["lse_out"]} if s["lse"] else {"out": out}
    if s["kind"] == "append":
        return {"q": plain_append(s), "k": s["k_cache"], "v": s["v_cache"]}
    out, lse = plain_decode(s) if s["kind"] == "decode" else plain_prompt(s)
    return {"out": out, "lse": lse} if s["lse"] else {"out": out}


def work(case):
    c = case
    Hq, Hkv, D = c["Hq"], c["Hkv"], c["D"]
    if c["kind"] == "append":
        # Every row of q, k and v read and written, a row of the table a token.
        return {"bytes": c["T"] * (4 * (Hq + 2 * Hkv) * D + 4 * c["rot"] + 8), "flops": c["T"] * 3 * (Hq + Hkv) * c["rot"]}
    if c["kind"] == "decode":
        n = sum(_decode_lengths(c))
        return {"bytes": 4 * Hkv * D * n + 4 * Hq * D * c["B"], "flops": 4 * Hq * D * n}
    new, keys = _prompt_lengths(c)
    pairs = sum(a * b - (a * (a - 1) // 2 if c["causal"] else 0) for a, b in zip(new, keys))
    return {"bytes": 4 * Hkv * D * sum(keys) + 4 * Hq * D * sum(new), "flops": 4 * Hq * D * pairs}


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

    k, v = s["k_cache"].double(), s["v_cache"].double()
    row = s["pages"].long()[s["seqs"].long(), at // c["page"]] * c["page"] + at % c["page"]
    k.flatten(0, 1)[row] = turned(s["k"])
    v.flatten(0, 1)[row] = s["v"].double()
    return {"q": turned(s["q"]), "k": k, "v": v}


def _softmax64(q, k, v, seen):
    """q [h, n, D], k and v [m, D], seen [n, m] or None, in 64 bits."""
    x = q @ k.T * (1.0 / math.sqrt(q.shape[-1]))
    if seen is not None:
        x = torch.where(seen, x, -math.inf)
    lse = torch.logsumexp(x, -1)
    return torch.exp(x - lse[..., None]) @ v, lse


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "append":
        return exact_append(c, s)
    # Sequence by sequence, kv head by kv head, a block of query rows at a time.
    new, keys = ([1] * c["B"], _decode_lengths(c)) if c["kind"] == "decode" else _prompt_lengths(c)
    G = c["Hq"] // c["Hkv"]
    out = torch.zeros((sum(new), c["Hq"], c["D"]), dtype=torch.float64, device="cuda")
    lse = torch.full((sum(new), c["Hq"]), -math.inf, dtype=torch.float64, device="cuda")
    at = 0
    for b, (n, m) in enumerate(zip(new, keys)):
        if c["page"]:
            used = s["pages"][b, :-(-m // c["page"])].long()
            k, v = (s[name][used].flatten(0, 1)[:m] for name in ("k_cache", "v_cache"))
        else:
            k, v = s["k"][at:at + m], s["v"][at:at + m]
        for h in range(c["Hkv"] if m else 0):
            kh, vh, heads = k[:, h].double(), v[:, h].double(), slice(h * G, (h + 1) * G)
            for r in range(0, n, 1024):
                e = min(n, r + 1024)
                seen = None
                if c.get("causal"):
                    seen = (torch.arange(r, e, device="cuda")[:, None] + (m - n) >= torch.arange(m, device="cuda")[None, :])
                o, z = _softmax64(s["q"][at + r:at + e, heads].transpose(0, 1).double(), kh, vh, seen)
                out[at + r:at + e, heads], lse[at + r:at + e, heads] = o.transpose(0, 1), z.T
        at += n
    return {"out": out, "lse": lse} if c["lse"] else {"out": out}
