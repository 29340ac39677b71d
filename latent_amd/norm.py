"""Between two blocks of a layer: norms before and after a block, with its gate and the residual stream, in one pass.

    residual_norm   x' = x + scale gate post(y),  n = pre(x')

y is what a block gave for the stream x, n what the next block reads.  The
reference leaves norms to llama.cpp's graph (README.md:111-113).
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from .attention import _attend, _on

_KINDS = {"rms": _lib.LATENT_NORM_RMS, "layer": _lib.LATENT_NORM_LAYER}
_DTYPES = {torch.float32: _lib.LATENT_F32, torch.float16: _lib.LATENT_F16, torch.bfloat16: _lib.LATENT_BF16}


class Norm:
    """A norm of rows of d numbers: kind "rms", v / sqrt(mean(v^2) + eps) weight + bias, or "layer", the same of v - mean(v).

    weight and bias: [d], f32, f16 or bf16 (both of one type), either None for ones and zeros.  All four may be set later on: a
    call takes them as they are then (a captured one has those of its capture).
    """

    __slots__ = ("weight", "bias", "_kind", "_eps")

    def __init__(self, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, kind: str = "rms", eps: float = 1e-6):
        self.weight, self.bias, self.kind, self.eps = weight, bias, kind, eps

    @property
    def kind(self) -> str:
        return self._kind

    @kind.setter
    def kind(self, kind: str) -> None:
        if kind not in _KINDS:
            raise ValueError(f"kind must be one of {sorted(_KINDS)}")
        self._kind = kind

    @property
    def eps(self) -> float:
        return self._eps

    @eps.setter
    def eps(self, eps: float) -> None:
        if not 0.0 <= eps < float("inf"):
            raise ValueError("eps must be finite and not negative")
        self._eps = float(eps)

    @property
    def _args(self):
        return _KINDS[self._kind], self._eps, self.weight, self.bias


class BlockNorm:
    """A block's place in the residual stream: it reads pre(x) and adds scale gate post(y); each of pre, post, gate may be None.

    gate: [d] (one for all tokens).  DecodeStack takes one for each of its blocks.
    """

    __slots__ = ("pre", "post", "gate", "scale")

    def __init__(self, pre: Optional[Norm] = None, post: Optional[Norm] = None, gate: Optional[torch.Tensor] = None, scale: float = 1.0):
        if gate is not None and gate.dim() != 1:
            raise ValueError("gate must be [d]")
        self.pre, self.post, self.gate, self.scale = pre, post, gate, float(scale)

    def add(self, x: torch.Tensor, y: torch.Tensor, following: "Optional[BlockNorm]", dtype: torch.dtype,
            x_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """The stream after the block gave y for it, and what the following block reads (the stream itself, where it has no pre)."""
        x, n = residual_norm(x, y, post=self.post, gate=self.gate, scale=self.scale, pre=None if following is None else following.pre,
                             dtype=dtype, x_out=x_out)
        return x, x if n is None else n


def residual_norm(
    x: torch.Tensor,
    y: Optional[torch.Tensor] = None,
    post: Optional[Norm] = None,
    gate: Optional[torch.Tensor] = None,
    scale: float = 1.0,
    pre: Optional[Norm] = None,
    dtype: Optional[torch.dtype] = None,
    x_out: Optional[torch.Tensor] = None,
    n_out: Optional[torch.Tensor] = None,
    stream: Optional[torch.cuda.Stream] = None,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """x' = x + scale gate post(y) and n = pre(x'), row by row: x, y [T, d] (d <= 32768), each f32, f16 or bf16.

    gate: [d], [T, 1] or [T, d]; post, gate: None for none.  Without y, x' is x
    itself; without pre there is no n (None).  x' has x's type, n dtype (default:
    x's); x_out may be x.  Sums are fp32, and n is taken from x' before x' is
    rounded to its type.  There is no backward pass.
    """
    if not (post is None or isinstance(post, Norm)) or not (pre is None or isinstance(pre, Norm)):
        raise TypeError("post and pre must be Norm")
    if not isinstance(x, torch.Tensor):
        raise TypeError("x must be a tensor")
    want = _DTYPES.get(x.dtype if dtype is None else dtype)
    if want is None:
        raise TypeError("x and dtype must be float32, float16 or bfloat16")
    args = (x, y, None if post is None else post._args, gate, scale, None if pre is None else pre._args, want, x_out, n_out)
    if stream is not None:
        with _on(stream, x):
            return _attend.residual_norm(*args)
    return _attend.residual_norm(*args)
