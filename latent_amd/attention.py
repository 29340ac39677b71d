"""The attention half of a decoder layer: a paged key-value cache and what reads and fills it.

    kv_append            a step's keys (rotated by their positions) and values into the
                         cache, its queries rotated in the same launch
    attend_decode        one new token a sequence over the cache
    attend_prompt        whole prompts, packed, causal
    attend_prompt_paged  the same with keys and values in the cache (a chunk of a
                         prompt behind the part that is cached)
    Attention            projections, cache and these calls as one block, which
                         DecodeStack puts before each layer's experts

The reference leaves attention to llama.cpp's graph (README.md:111-113).

A cache is a pair of tensors [pages, page rows, kv heads, D], f16 or bf16 (any
strides that are multiples of 8 elements, D adjacent: permuted views work), with
a page table int32 [B, max_pages]: position p of sequence b is row p % page of
page pages[b, p // page].  A page id outside [0, pages) names no page.  Query
head h reads kv head h // (n_head / n_kv_head).  D is a multiple of 8 up to 256.
Scores, softmax and sums are fp32 (a row's sum of values times weights of at most
one has to stay finite there); probabilities are rounded to the element type
for the product with the values, outputs once.  There is no backward pass.
Lengths are cut off at what a row of the page table has room for, and at 0.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from . import _lib
from ._lib import LatentAttnDecodeArgs, LatentAttnPromptArgs, LatentError, LatentKvCache, check, lib


class _NoBinding:
    """In the binding's place where it cannot be loaded: the rest of the package works, an attention call raises."""

    def __init__(self, cause: ImportError):
        self._cause = cause

    def __getattr__(self, name: str):
        raise ImportError("latent_amd/_attend.so is missing or does not fit this torch: build it with "
                          f"`python latent_amd/build.py` ({self._cause})") from self._cause


try:
    from . import _attend
except ImportError as e:
    _attend = _NoBinding(e)
else:
    _attend.entries(*(ctypes.cast(lib[f"latent_{n}"], ctypes.c_void_p).value for n in (
        "kv_append", "attn_decode_workspace_size", "attn_decode", "attn_prompt_workspace_size", "attn_prompt")), LatentError)

_DTYPE = (torch.float16, torch.bfloat16)


def _on(stream: torch.cuda.Stream, t: torch.Tensor):
    if t.device != stream.device:
        raise ValueError(f"a stream of {stream.device} for tensors on {t.device}")
    return torch.cuda.stream(stream)


def rope_table(n_positions: int, rot_dim: int, base: float = 10000.0, device="cuda") -> torch.Tensor:
    """cos and sin of position p times base^(-2i / rot_dim), f32 [n_positions, 2, rot_dim / 2]
    (angles in 64 bits: in 32 a far position's angle is off by more than the table's rounding)."""
    if n_positions < 0 or rot_dim <= 0 or rot_dim % 2:
        raise ValueError("rot_dim must be even and positive")
    i = torch.arange(0, rot_dim, 2, dtype=torch.float64, device=device)
    angle = torch.arange(n_positions, dtype=torch.float64, device=device)[:, None] * base ** (-i / rot_dim)
    return torch.stack((angle.cos(), angle.sin()), 1).float().contiguous()


def kv_append(
    k: torch.Tensor,
    v: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    pages: torch.Tensor,
    positions: torch.Tensor,
    seqs: Optional[torch.Tensor] = None,
    q: Optional[torch.Tensor] = None,
    rope: Optional[torch.Tensor] = None,
    interleaved: bool = False,
    q_out: Optional[torch.Tensor] = None,
    stream: Optional[torch.cuda.Stream] = None,
) -> Optional[torch.Tensor]:
    """Stores keys and values [T, kv heads, D] in the cache, keys rotated; returns q rotated (None without q).

    Token t belongs to sequence seqs[t] (int32 [T]; t itself when None) at
    positions[t].  rope: f32 [positions, 2, rot / 2] cos and sin (rope_table);
    the leading rot of D dimensions turn, dimension i with i + rot / 2, or
    neighbours when `interleaved`.  None: nothing is rotated.  q_out may be q.
    A token whose position is negative or beyond the table is left out, q_out
    row and all; one whose sequence or page does not exist is not stored.
    Tokens of one call must not name the same cache row twice: what it holds
    then is unspecified.
    """
    if stream is not None:
        with _on(stream, k):
            return _attend.kv_append(k, v, k_cache, v_cache, pages, positions, seqs, q, rope, interleaved, q_out)
    return _attend.kv_append(k, v, k_cache, v_cache, pages, positions, seqs, q, rope, interleaved, q_out)


def attend_decode(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    pages: torch.Tensor,
    lengths: torch.Tensor,
    scale: Optional[float] = None,
    out: Optional[torch.Tensor] = None,
    lse: Optional[torch.Tensor] = None,
    workspace: Optional[torch.Tensor] = None,
    stream: Optional[torch.cuda.Stream] = None,
) -> torch.Tensor:
    """One new token a sequence: q [B, heads, D] over the first lengths[b] (int32 [B]) positions of the cache.

    scale defaults to D^-0.5.  A row without keys (length 0, or only on pages
    that do not exist) gives zeros.  lse: f32 [B, heads], filled with the log
    of the sum of exp(scale q . k) (-inf without keys), as joining the results
    of several caches needs it.  A workspace that is given
    (attend_decode_workspace_size bytes) must not serve calls that may overlap.
    """
    if stream is not None:
        with _on(stream, q):
            return _attend.attend_decode(q, k_cache, v_cache, pages, lengths, scale, out, lse, workspace)
    return _attend.attend_decode(q, k_cache, v_cache, pages, lengths, scale, out, lse, workspace)


def attend_decode_workspace_size(n_seq: int, n_head: int, n_kv_head: int, head_dim: int, max_pages: int, page_size: int) -> int:
    """Workspace bytes of attend_decode for these sizes."""
    cache = LatentKvCache(n_pages=1, page_size=page_size, n_seq=n_seq, max_pages=max_pages, pages_stride=max_pages)
    a = LatentAttnDecodeArgs(cache=cache, n_head=n_head, n_kv_head=n_kv_head, head_dim=head_dim, dtype=_lib.LATENT_BF16, scale=1.0)
    n = ctypes.c_size_t()
    check(lib.latent_attn_decode_workspace_size(ctypes.byref(a), ctypes.byref(n)), "latent_attn_decode_workspace_size")
    return int(n.value)


def attend_prompt_workspace_size(n_tokens: int, n_seq: int, n_head: int, n_kv_head: int, head_dim: int, n_keys: int = 0,
                                 max_pages: int = 0, page_size: int = 1) -> int:
    """Workspace bytes of attend_prompt (n_keys rows of keys) or attend_prompt_paged for these sizes; 0: it takes none."""
    cache = LatentKvCache(n_pages=1, page_size=page_size, n_seq=n_seq, max_pages=0 if n_keys else max_pages,
                          pages_stride=max_pages)
    a = LatentAttnPromptArgs(cache=cache, n_tokens=n_tokens, n_keys=n_keys, n_head=n_head, n_kv_head=n_kv_head,
                             head_dim=head_dim, dtype=_lib.LATENT_BF16, causal=1, scale=1.0)
    n = ctypes.c_size_t()
    check(lib.latent_attn_prompt_workspace_size(ctypes.byref(a), ctypes.byref(n)), "latent_attn_prompt_workspace_size")
    return int(n.value)


def attend_prompt(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    starts: torch.Tensor,
    k_starts: Optional[torch.Tensor] = None,
    causal: bool = True,
    scale: Optional[float] = None,
    out: Optional[torch.Tensor] = None,
    lse: Optional[torch.Tensor] = None,
    workspace: Optional[torch.Tensor] = None,
    stream: Optional[torch.cuda.Stream] = None,
) -> torch.Tensor:
    """Whole prompts, packed: sequence b is rows starts[b] .. starts[b + 1] - 1 (int32 [B + 1], ascending) of
    q [T, heads, D] and of k, v [Tk, kv heads, D] (rows k_starts[b] .. where k_starts is given).

    Causal with the ends aligned: with n queries and m keys, query i sees keys
    j <= i + m - n.  Rows of out and lse (f32 [T, heads]) that belong to no
    sequence are not written; a row that sees no key is zeros, lse -inf.
    A workspace that is given (attend_prompt_workspace_size bytes, fewer: the
    call does without) must not serve calls that may overlap.
    """
    if stream is not None:
        with _on(stream, q):
            return _attend.attend_prompt(q, k, v, starts, k_starts, causal, scale, out, lse, workspace)
    return _attend.attend_prompt(q, k, v, starts, k_starts, causal, scale, out, lse, workspace)


def attend_prompt_paged(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    pages: torch.Tensor,
    lengths: torch.Tensor,
    starts: torch.Tensor,
    causal: bool = True,
    scale: Optional[float] = None,
    out: Optional[torch.Tensor] = None,
    lse: Optional[torch.Tensor] = None,
    workspace: Optional[torch.Tensor] = None,
    stream: Optional[torch.cuda.Stream] = None,
) -> torch.Tensor:
    """attend_prompt with the keys and values of sequence b in the cache: its first lengths[b] (int32 [B])
    positions, the new tokens' own (appended before the call) the last of them.  lengths[b] is at most what a row of
    pages has room for: what is beyond is cut off, and the last query then stands at the last position that is left."""
    if stream is not None:
        with _on(stream, q):
            return _attend.attend_prompt_paged(q, k_cache, v_cache, pages, lengths, starts, causal, scale, out, lse, workspace)
    return _attend.attend_prompt_paged(q, k_cache, v_cache, pages, lengths, starts, causal, scale, out, lse, workspace)


class Attention:
    """One layer's attention: projections, a paged cache of its own, and the calls above.

    w_qkv [d, (n_head + 2 n_kv_head) D] holds the columns of q, k and v one after
    the other, w_o [n_head D, d] the output projection; both f16 or bf16, the
    cache's type too.  The cache has n_pages pages of page_size positions; which
    sequence owns which page is the caller's, in the page table of each call.
    """

    def __init__(self, w_qkv: torch.Tensor, w_o: torch.Tensor, n_head: int, n_kv_head: int, n_pages: int, page_size: int,
                 rope: Optional[torch.Tensor] = None, interleaved: bool = False, scale: Optional[float] = None):
        if w_qkv.dim() != 2 or w_o.dim() != 2 or w_qkv.dtype not in _DTYPE or w_o.dtype != w_qkv.dtype or not w_qkv.is_cuda:
            raise TypeError("w_qkv and w_o must be CUDA f16 or bf16 matrices")
        if n_head <= 0 or n_kv_head <= 0 or n_head % n_kv_head or w_o.shape[0] % n_head:
            raise ValueError("n_head must be a multiple of n_kv_head, and w_o's rows one of n_head")
        D = w_o.shape[0] // n_head
        if D % 8 or not 0 < D <= 256:
            raise ValueError(f"heads of {D} dimensions: a multiple of 8 up to 256 is supported")
        if w_qkv.shape[1] != (n_head + 2 * n_kv_head) * D or w_o.shape[1] != w_qkv.shape[0] or w_o.device != w_qkv.device:
            raise ValueError(f"w_qkv {list(w_qkv.shape)} and w_o {list(w_o.shape)} do not fit {n_head} and {n_kv_head} heads")
        self.w_qkv, self.w_o = w_qkv.detach().contiguous(), w_o.detach().contiguous()
        self.n_head, self.n_kv_head, self.head_dim = int(n_head), int(n_kv_head), int(D)
        self.rope, self.interleaved, self.scale = rope, bool(interleaved), scale
        shape = (int(n_pages), int(page_size), self.n_kv_head, self.head_dim)
        self.k_cache, self.v_cache = (torch.zeros(shape, dtype=w_qkv.dtype, device=w_qkv.device) for _ in range(2))

    @property
    def n_embd(self) -> int:
        return int(self.w_qkv.shape[0])

    def _append(self, x: torch.Tensor, pages, positions, seqs) -> torch.Tensor:
        H, K = self.n_head, self.n_kv_head
        qkv = (x.to(self.w_qkv.dtype) @ self.w_qkv).view(x.shape[0], H + 2 * K, self.head_dim)
        q = qkv[:, :H]
        return kv_append(qkv[:, H:H + K], qkv[:, H + K:], self.k_cache, self.v_cache, pages, positions, seqs=seqs,
                         q=q, rope=self.rope, interleaved=self.interleaved, q_out=q)

    def _stored_limit(self, max_pages: int) -> Optional[int]:
        """How many positions tokens are stored at, where the rotation table ends before a page table row of max_pages does
        (else None).  A token behind it is left out of the cache and its query is not rotated, so its attention is zeros: a
        launch or two more, which a table of as many positions as the pages spares."""
        if self.rope is None or self.rope.shape[0] >= max_pages * self.k_cache.shape[1]:
            return None
        return int(self.rope.shape[0])

    def _project(self, a: torch.Tensor) -> torch.Tensor:
        return a.view(a.shape[0], self.w_o.shape[0]) @ self.w_o

    def decode(self, x: torch.Tensor, pages: torch.Tensor, positions: torch.Tensor, lengths: torch.Tensor,
               workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
        """One new token a sequence: x [B, d] at positions [B]; lengths [B] count it.  Returns [B, d] in the weights' type.
        A token behind the rotation table is not stored, and its attention is zeros."""
        q = self._append(x, pages, positions, None)
        limit = self._stored_limit(pages.shape[1])
        if limit is not None:
            lengths = lengths.masked_fill(positions >= limit, 0)
        return self._project(attend_decode(q, self.k_cache, self.v_cache, pages, lengths, scale=self.scale, workspace=workspace))

    def prompt(self, x: torch.Tensor, pages: torch.Tensor, positions: torch.Tensor, seqs: torch.Tensor, starts: torch.Tensor,
               lengths: torch.Tensor) -> torch.Tensor:
        """New tokens of several sequences, packed: x [T, d], token t of sequence seqs[t] (row of pages) at positions[t],
        sequence b's being rows starts[b] .. starts[b + 1] - 1 and the last of its lengths[b].  Rows of no sequence
        (padding, at negative positions) and tokens behind the rotation table, which are not stored, give zeros; the pages
        have to have room for lengths[b]."""
        q = self._append(x, pages, positions, seqs)
        out = torch.zeros_like(q, memory_format=torch.contiguous_format)
        attend_prompt_paged(q, self.k_cache, self.v_cache, pages, lengths, starts, scale=self.scale, out=out)
        limit = self._stored_limit(pages.shape[1])
        if limit is not None:  # only these rows see what was not stored: the others' positions are in front of it
            out.masked_fill_((positions >= limit)[:, None, None], 0)
        return self._project(out)
