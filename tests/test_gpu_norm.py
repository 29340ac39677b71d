"""residual_norm on the GPU against 64 bits.

Sums of d squares in fp32, a lane's in order and the lanes' in a tree: no more than (d / 512 + 40) roundings of 2^-24 deep for
the sizes here; the root halves them, and what is left (a division, a root, four products and sums) is within 16 more.
A layer norm's mean is off by as many roundings of the row's largest number, before the squares see it.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
W = 2.0 ** -24


@pytest.fixture(scope="module")
def la(gpu):
    return gpu


def normed64(v, n, err):
    """n of v (f64) whose elements are off by err, and how far the result may be."""
    if n is None:
        return v, err
    d = v.shape[-1]
    depth = (d / 512 + 40) * W
    u = v
    if n.kind == "layer":
        u = v - v.mean(-1, keepdim=True)
        err = err + err.mean(-1, keepdim=True) + depth * v.abs().amax(-1, keepdim=True)
    r = (u.square().mean(-1, keepdim=True) + n.eps).rsqrt()
    # d(u r) = r du + u dr, |dr| <= r^3 mean(|u| |du|)
    off = r * err + u.abs() * (r ** 3 * (u.abs() * err).mean(-1, keepdim=True) + r * (depth + 16 * W))
    w = 1.0 if n.weight is None else n.weight.double()
    b = torch.zeros(()).cuda().double() if n.bias is None else n.bias.double()
    got = u * r * w + b
    return got, off * abs(w) + 4 * W * (got.abs() + b.abs())


def reference(x, y, post, gate, scale, pre):
    x = x.double()
    err = torch.zeros_like(x)
    if y is not None:
        z, off = normed64(y.double(), post, torch.zeros_like(x))
        g = 1.0 if gate is None else gate.double()
        z, off = z * g * scale, off * abs(g) * abs(scale)
        x, err = x + z, off + 4 * W * (z.abs() + (x + z).abs())
    return (x, err), normed64(x, pre, err)


def near(got, want, err):
    u = torch.finfo(got.dtype).eps / 2
    off = (got.double() - want).abs() - err * 1.01 - u * (want.abs() + err) - torch.finfo(got.dtype).smallest_normal
    assert float(off.max()) <= 0, f"off by {float(off.max())} too much"


def norm(la, g, d, kind, dt, bias):
    if kind is None:
        return None
    w = (1 + 0.3 * torch.randn(d, generator=g, device="cuda")).to(dt) if bias != "bare" else None
    b = torch.randn(d, generator=g, device="cuda").to(dt) if bias is True else None
    return la.Norm(w, bias=b, kind=kind, eps=1e-5)


@pytest.mark.parametrize("rows,d", [(1, 1), (3, 7), (5, 64), (2, 513), (9, 1000), (6, 1024), (3, 2048), (2, 2056), (1, 4096), (5, 4100), (3, 7168), (2, 8192), (2, 8200),
                                    (1, 16384), (2, 16391), (1, 32768), (300, 384), (1100, 2048)])
@pytest.mark.parametrize("x,y,n,post,pre,gate", [
    ("f32", "bf16", "bf16", "rms", "rms", "row"), ("bf16", "f32", "f32", "layer", "layer", "all"), ("f16", "f16", "f16", None, "rms", None),
    ("f32", None, "f16", None, "layer", None), ("f32", "f32", "bf16", "rms", None, "token")])
def test_against_64_bits(la, rows, d, x, y, n, post, pre, gate):
    g = torch.Generator(device="cuda").manual_seed(rows * d)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    xt = (3 * r(rows, d) + 1).to(T[x])
    yt = None if y is None else (r(rows, d) * torch.exp2(2 * r(rows, 1)) - 0.5).to(T[y])
    post, pre = norm(la, g, d, post, T[x], x == "bf16"), norm(la, g, d, pre, torch.float32, True if x == "f32" else "bare")
    gt = None if gate is None else {"row": r(d), "all": r(rows, d).to(T[x]), "token": r(rows, 1)}[gate]
    xo, no = la.residual_norm(xt, yt, post=post, gate=gt, scale=0.7, pre=pre, dtype=T[n])
    (wx, ex), (wn, en) = reference(xt, yt, post, gt, 0.7, pre)
    if y is None:
        assert xo is xt
    near(xo, wx, ex)
    if pre is None:
        assert no is None
    else:
        assert no.dtype == T[n]
        near(no, wn, en)


def test_in_place_strides_and_given_outputs(la):
    g = torch.Generator(device="cuda").manual_seed(3)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    pre, post = la.Norm(r(200).bfloat16()), la.Norm(r(200))
    big, y = r(7, 3, 200), r(200, 7).t()  # rows apart; columns apart (copied)
    x = big[:, 1]
    want, n = la.residual_norm(x.clone(), y.contiguous(), post=post, pre=pre, dtype=torch.float16)
    others, n_big = big[:, ::2].clone(), torch.full((9, 264), 5.0, dtype=torch.float16, device="cuda")
    xo, no = la.residual_norm(x, y, post=post, pre=pre, dtype=torch.float16, x_out=x, n_out=n_big[1:8, 8:208])
    assert xo is x and torch.equal(x, want) and torch.equal(big[:, ::2], others) and torch.equal(no, n)
    n_big[1:8, 8:208] = 5.0
    assert bool((n_big == 5.0).all())
    odd = r(3, 211)[:, 3:203]  # 16 bytes do not divide the base: other sums, each as far from the exact one as reference() has it
    xo, no = la.residual_norm(odd, y[:3], post=post, pre=pre)
    (wx, ex), (wn, en) = reference(odd, y[:3], post, None, 1.0, pre)
    near(xo, wx, ex)
    near(no, wn, en)


def test_rows_of_zeros_and_rows_that_are_not_finite(la):
    x = torch.zeros((4, 1024), device="cuda")
    x[1, 3], x[2, 1000] = math.inf, math.nan
    x[3] = 1e-30
    _, n = la.residual_norm(x, pre=la.Norm(eps=0.0))
    assert bool(torch.isnan(n[0]).all()) and bool(torch.isnan(n[1, 3])) and bool(torch.isnan(n[2]).all())
    _, n = la.residual_norm(x, pre=la.Norm(eps=1e-6))
    assert bool((n[0] == 0).all()) and bool(torch.isfinite(n[3]).all())
    y = torch.zeros_like(x)
    xo, _ = la.residual_norm(torch.ones_like(x), y, post=la.Norm(kind="layer"))
    assert bool((xo == 1).all())


@pytest.mark.parametrize("rows,d", [(0, 8), (4, 0), (0, 0)])
def test_nothing_to_do(la, rows, d):
    x = torch.zeros((rows, d), device="cuda")
    xo, n = la.residual_norm(x, x.clone(), pre=la.Norm(torch.ones(d, device="cuda")), dtype=torch.bfloat16)
    assert xo.shape == n.shape == (rows, d) and n.dtype == torch.bfloat16
