"""residual_norm's operands as a program changes and broadcasts them, against 64 bits (tests/test_gpu_norm.py's bounds)."""

import pytest
import torch

from tests.test_gpu_norm import near, reference

pytestmark = pytest.mark.gpu


def test_a_norm_that_is_changed_between_calls(gpu):
    g = torch.Generator(device="cuda").manual_seed(1)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    x, y = r(5, 384), r(5, 384)
    n = gpu.Norm(r(384), eps=1e-5)
    for change in (dict(), dict(weight=r(384)), dict(bias=r(384)), dict(kind="layer"), dict(eps=0.5), dict(weight=None, bias=r(384).bfloat16()), dict(bias=None)):
        for name, value in change.items():
            setattr(n, name, value)
        xo, no = gpu.residual_norm(x, y, post=n, pre=n)
        (wx, ex), (wn, en) = reference(x, y, n, None, 1.0, n)
        near(xo, wx, ex)
        near(no, wn, en)


@pytest.mark.parametrize("gate", ["row", "all", "token", None])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("d", [96, 100, 2056])
def test_broadcast_operands_have_their_rows_values(gpu, d, kind, gate):
    """x and y with a row stride of zero, a post norm of a bias alone, gates of each form and of another type."""
    g = torch.Generator(device="cuda").manual_seed(d)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    T = 5
    x, y = r(1, d).expand(T, d), r(1, d).half().expand(T, d)
    gt = {"row": r(d), "all": r(T, d), "token": r(T, 1), None: None}[gate]
    gt = gt if gt is None else gt.bfloat16()
    post, pre = gpu.Norm(bias=r(d), kind=kind, eps=1e-5), gpu.Norm(kind="layer", eps=1e-5)
    xo, no = gpu.residual_norm(x, y, post=post, gate=gt, scale=-1.5, pre=pre, dtype=torch.float16)
    (wx, ex), (wn, en) = reference(x, y, post, gt, -1.5, pre)
    near(xo, wx, ex)
    near(no, wn, en)
    again = gpu.residual_norm(x.contiguous(), y.contiguous(), post=post, gate=gt if gate != "token" else gt.expand(T, d).contiguous(), scale=-1.5, pre=pre,
                              dtype=torch.float16)
    assert torch.equal(xo, again[0]) and torch.equal(no, again[1])
    if gate in ("all", "token"):
        assert not torch.equal(xo[0], xo[1])


def test_an_output_of_one_row_for_all_is_refused(gpu):
    x = torch.zeros((5, 96), device="cuda")
    for name in ("x_out", "n_out"):
        with pytest.raises(ValueError):
            gpu.residual_norm(x, x, pre=gpu.Norm(), **{name: torch.zeros((1, 96), device="cuda").expand(5, 96)})
