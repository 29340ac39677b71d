"""8-bit caches for tests: the format in plain torch operations, and caches whose unused rows would spoil a result.

Codes and scales are elementwise operations of fp32 (a maximum, a reciprocal, a division, two products, a rounding), each
rounded by itself, so the kernel's have to be the same to the bit.  What attention reads is code times
scale, in 64 bits; tests/_attention.py's tolerances then hold as they are: a score's scale is one more
rounding than the D products and their sum (it counts D + 4), a probability's two more of the 4 w there, and
the probability times its value's scale is what is rounded to the element type.
"""

from __future__ import annotations

import torch

CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
LEAST = 2.0 ** -100


def quantise(x, code):
    """Codes and scales [..., D] -> codes [..., D], scale [...]."""
    x = x.float()
    most = x.abs().amax(-1)
    finite = torch.isfinite(x).all(-1)
    m = torch.where(finite, most, 0.0).clamp(min=LEAST)
    top = torch.full_like(m, TOP[code])  # a tensor: torch divides by a number through its reciprocal
    y = torch.where(finite[..., None], x, 0.0) * (top * m.reciprocal())[..., None]
    scale = torch.where(finite, m / top, float("nan"))
    return (y.round() if code == torch.int8 else y).to(code), scale


def values(codes, scale):
    """What codes and scales stand for, f64."""
    return codes.float().double() * scale.double()[..., None]


def bits(t):
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


def take(cache, *index):
    """cache[index] (torch indexes no 8-bit floating point)."""
    return bits(cache)[index].view(cache.dtype)


def put(cache, index, codes):
    bits(cache)[index] = bits(codes)


def empty_cache(n, page, Hkv, D, code, fill=0x7F, order="rows"):
    """Codes of `fill` (e4m3's NaN) and scales of NaN."""
    shape = (n, page, Hkv, D) if order == "rows" else (n, Hkv, page, D)
    c = torch.full(shape, fill, dtype=torch.uint8, device="cuda").view(code)
    c = c if order == "rows" else c.transpose(1, 2)
    return c, torch.full((n, Hkv, page), float("nan"), device="cuda")


def paged8(gen, lengths, page, Hkv, D, dt, code, spare=3, width=None, order="rows", shared=0):
    """(k_cache, v_cache, k_scale, v_scale, pages, [(k, v) of each sequence, f64]); the first `shared` pages are every sequence's."""
    need = [max(-(-n // page), shared) for n in lengths]
    width = max(need + [1]) if width is None else width
    total = shared + sum(n - shared for n in need) + spare
    perm = torch.randperm(total, generator=gen, device="cuda").int()
    table = torch.full((len(lengths), width), -1, dtype=torch.int32, device="cuda")
    kc, ks = empty_cache(total, page, Hkv, D, code, order=order)
    vc, vs = empty_cache(total, page, Hkv, D, code, order=order)

    def fill(ids, n):
        """Rows for the n positions of these pages."""
        got = []
        p = torch.arange(n, device="cuda")
        rows = ids.long()[p // page]
        for c, s in ((kc, ks), (vc, vs)):
            x = torch.randn((n, Hkv, D), generator=gen, device="cuda").to(dt)
            x *= torch.exp2(torch.randint(-3, 4, (n, Hkv, 1), generator=gen, device="cuda").float()).to(dt)
            codes, scale = quantise(x, code)
            put(c, (rows, p % page), codes)
            s[rows, :, p % page] = scale
            got.append(values(codes, scale))
        return got

    common = fill(perm[:shared], shared * page) if shared else None
    seqs, at = [], shared
    for b, n in enumerate(lengths):
        ids = torch.cat((perm[:shared], perm[at:at + need[b] - shared]))
        at += need[b] - shared
        table[b, :need[b]] = ids
        own = fill(ids[shared:], max(0, n - shared * page))
        seqs.append(tuple((torch.cat((c, o)) if shared else o)[:n] for c, o in zip(common or own, own)))
    return kc, vc, ks, vs, table, seqs
