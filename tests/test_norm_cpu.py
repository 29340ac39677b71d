"""What residual_norm hands to the library, where no GPU is needed to see it."""

import math

import pytest
import torch

import latent_amd
from latent_amd import _lib, norm


@pytest.fixture
def handed(monkeypatch):
    """The arguments of each call of the binding."""
    calls = []

    class Binding:
        def residual_norm(self, *args):
            calls.append(args)
            return args[0], args[0]

    monkeypatch.setattr(norm, "_attend", Binding())
    return calls


def test_a_norms_attributes_are_those_of_the_call(handed):
    x, w, b = torch.zeros(2, 4), torch.full((4,), 2.0), torch.full((4,), 3.0)
    n = latent_amd.Norm(torch.ones(4))
    block = latent_amd.BlockNorm(pre=n, post=n)
    latent_amd.residual_norm(x, pre=n)
    n.weight, n.bias, n.kind, n.eps = w, b, "layer", 0.5
    latent_amd.residual_norm(x, x, post=n, pre=n)
    block.add(x, x, block, torch.float32)
    n.weight = n.bias = None
    latent_amd.residual_norm(x, pre=n)
    first, second, third, last = handed
    assert first[5][:2] == (_lib.LATENT_NORM_RMS, 1e-6) and bool((first[5][2] == 1).all()) and first[5][3] is None
    for post, pre in ((second[2], second[5]), (third[2], third[5])):
        for got in (post, pre):
            assert got[:2] == (_lib.LATENT_NORM_LAYER, 0.5) and got[2] is w and got[3] is b
    assert last[5] == (_lib.LATENT_NORM_LAYER, 0.5, None, None)


@pytest.mark.parametrize("name,value", [("kind", "batch"), ("kind", None), ("eps", -1.0), ("eps", math.nan), ("eps", math.inf)])
def test_attributes_that_no_norm_has_are_refused(handed, name, value):
    n = latent_amd.Norm()
    with pytest.raises(ValueError):
        setattr(n, name, value)
        latent_amd.residual_norm(torch.zeros(2, 4), pre=n)
    with pytest.raises(ValueError):
        latent_amd.Norm(**{name: value})
    assert not handed
