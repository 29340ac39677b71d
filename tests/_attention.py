"""Plain attention in 64 bits, and how far a kernel's result may be from it.

A result is off by what these roundings allow (u: half a step of the element
type, w = 2^-24 of fp32):
  - a score is a sum of D products that are exact in fp32:
        ds = (D + 4) w scale sum_d |q_d k_d| (sum, scaling, and the difference to the maximum)
    an error ds of a score changes its probability by the factor exp(+-ds);
  - exp2 and the sums over n keys, in blocks: (n + 64) w of the sum of what is added,
    doubled because numerator and sum both have it;
  - a probability is rounded to the element type for the product with v: u;
  - the output is rounded once: u |out|.
"""

from __future__ import annotations

import math

import torch

W = 2.0 ** -24


def half_step(dt: torch.dtype) -> float:
    return torch.finfo(dt).eps / 2


def attend64(q, k, v, seen, scale):
    """q [n, H, D], k and v [m, Hkv, D], seen bool [n, m] -> out, lse, tolerances of out and of lse (f64)."""
    n, H, D = q.shape
    m, Hkv = k.shape[:2]
    G = H // Hkv
    q, k, v = q.double(), k.double(), v.double()
    out = torch.zeros((n, H, D), dtype=torch.float64, device=q.device)
    lse = torch.full((n, H), -math.inf, dtype=torch.float64, device=q.device)
    tol, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
    if m == 0 or n == 0:
        return out, lse, tol, tol_lse
    any_seen = seen.any(1)
    for h in range(H):
        qh, kh = q[:, h], k[:, h // G]
        vh = v[:, h // G]
        x = torch.where(seen, scale * (qh @ kh.T), -math.inf)
        z = torch.logsumexp(x, 1)
        p = torch.where(seen, torch.exp(x - torch.where(any_seen, z, 0.0)[:, None]), 0.0)
        clean = torch.where(torch.isfinite(vh), vh, 0.0)
        o = p @ clean
        if not torch.isfinite(vh).all():  # only rows that see such a value get it
            bad = (seen.double() @ (~torch.isfinite(vh)).double()) > 0
            o = torch.where(bad, math.nan, o)
        out[:, h] = torch.where(any_seen[:, None], o, 0.0)
        lse[:, h] = torch.where(any_seen, z, -math.inf)
        size = torch.where(seen, scale * (qh.abs() @ kh.abs().T), 0.0).amax(1)
        ds = (D + 4) * W * size
        rest = 2 * (m + 64) * W
        tol[:, h] = (p @ clean.abs()) * (2 * ds + rest + 4 * W)[:, None]
        tol_lse[:, h] = ds + rest + 8 * W * (lse[:, h].abs() + 1)
    return out, lse, tol, tol_lse


def weight64(q, k, v, seen, scale):
    """sum_j p_j |v_j|, what the rounding of the probabilities is relative to."""
    finite = torch.where(torch.isfinite(v.double()), v.double().abs(), 0.0)
    return attend64(q, k, finite, seen, scale)[0]


def visible(n, m, causal, device):
    i, j = torch.arange(n, device=device)[:, None], torch.arange(m, device=device)[None, :]
    return (j <= i + (m - n)) if causal else torch.ones((n, m), dtype=torch.bool, device=device)


def assert_attention(got, got_lse, q, k, v, seen, scale):
    want, lse, tol, tol_lse = attend64(q, k, v, seen, scale)
    u = half_step(q.dtype)
    tol = tol + u * weight64(q, k, v, seen, scale) + u * want.abs() + torch.finfo(q.dtype).smallest_normal
    bad = torch.isnan(want)
    assert torch.equal(~torch.isfinite(got.double()), bad)
    off = torch.where(bad, 0.0, (got.double() - want).abs() - tol)
    assert float(off.max()) <= 0 if off.numel() else True, f"off by {float(off.max())} more than {float(tol.max())}"
    if got_lse is not None:
        assert torch.equal(torch.isinf(got_lse), torch.isinf(lse))
        d = torch.where(torch.isinf(lse), 0.0, (got_lse.double() - lse).abs() - tol_lse)
        assert float(d.max()) <= 0 if d.numel() else True, f"lse off by {float(d.max())} too much"


def paged(gen, lengths, page, Hkv, D, dt, spare=3, width=None, fill=float("nan"), order="rows"):
    """A cache whose unused rows hold `fill`: (k_cache, v_cache, pages, [(k, v) of each sequence])."""
    need = [-(-n // page) for n in lengths]
    width = max(need + [1]) if width is None else width
    total = sum(need) + spare
    perm = torch.randperm(total, generator=gen, device="cuda").int()
    table = torch.full((len(lengths), width), -1, dtype=torch.int32, device="cuda")
    shape = (total, page, Hkv, D) if order == "rows" else (total, Hkv, page, D)
    kc, vc = (torch.full(shape, fill, dtype=dt, device="cuda") for _ in range(2))
    if order != "rows":
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    seqs, at = [], 0
    for b, n in enumerate(lengths):
        table[b, :need[b]] = perm[at:at + need[b]]
        at += need[b]
        k, v = (torch.randn((n, Hkv, D), generator=gen, device="cuda").to(dt) for _ in range(2))
        p = torch.arange(n, device="cuda")
        rows = table[b].long()[p // page]
        kc[rows, p % page], vc[rows, p % page] = k, v
        seqs.append((k, v))
    return kc, vc, table, seqs
