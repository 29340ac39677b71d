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
Scores, softmax and sums are fp32; probabilities are rounded to the element type
for the product with the values, outputs once.  There is no backward pass.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import LatentAttnDecodeArgs, LatentAttnPromptArgs, LatentKvAppendArgs, LatentKvCache, check, lib

_DTYPE = {torch.float16: _lib.LATENT_F16, torch.bfloat16: _lib.LATENT_BF16}


def rope_table(n_positions: int, rot_dim: int, base: float = 10000.0, device="cuda") -> torch.Tensor:
    """cos and sin of position p times base^(-2i / rot_dim), f32 [n_positions, 2, rot_dim / 2]
    (angles in 64 bits: in 32 a far position's angle is off by more than the table's rounding)."""
    if n_positions < 0 or rot_dim <= 0 or rot_dim % 2:
        raise ValueError("rot_dim must be even and positive")
    i = torch.arange(0, rot_dim, 2, dtype=torch.float64, device=device)
    angle = torch.arange(n_positions, dtype=torch.float64, device=device)[:, None] * base ** (-i / rot_dim)
    return torch.stack((angle.cos(), angle.sin()), 1).float().contiguous()


def _heads(t: torch.Tensor, name: str, dt: torch.dtype, dev: torch.device) -> torch.Tensor:
    """[T, heads, D] as the kernels read it: a copy where the strides or the base do not fit."""
    if t.dim() != 3:
        raise ValueError(f"{name} must be [tokens, heads, D]")
    if t.dtype != dt:
        raise TypeError(f"{name} must be {dt}, as the queries and the cache are")
    if t.device != dev:
        raise ValueError(f"{name} must be on {dev}")
    st, sh, sd = t.stride()
    if (sd != 1 and t.shape[2] > 1) or st % 8 or sh % 8 or t.data_ptr() % 16:
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
    return t


def _ints(t: torch.Tensor, name: str, shape: Tuple[int, ...], dev: torch.device) -> torch.Tensor:
    if t.dtype != torch.int32 or tuple(t.shape) != shape or t.device != dev:
        raise ValueError(f"{name} must be int32 {list(shape)} on {dev}")
    return t if t.is_contiguous() else t.contiguous()


def _out(t: Optional[torch.Tensor], like: torch.Tensor, name: str) -> torch.Tensor:
    if t is None:
        return torch.empty(like.shape, dtype=like.dtype, device=like.device)
    if t.shape != like.shape or t.dtype != like.dtype or t.device != like.device:
        raise ValueError(f"{name} must be {like.dtype} {list(like.shape)} on {like.device}")
    st, sh, sd = t.stride()
    if (sd != 1 and t.shape[2] > 1) or st % 8 or sh % 8 or t.data_ptr() % 16:
        raise ValueError(f"{name} must have adjacent D, strides that are multiples of 8 and a 16-byte aligned base")
    return t


def _lse(t: Optional[torch.Tensor], T: int, Hq: int, dev: torch.device) -> int:
    if t is None:
        return 0
    if t.dtype != torch.float32 or tuple(t.shape) != (T, Hq) or t.device != dev or not t.is_contiguous():
        raise ValueError(f"lse must be contiguous f32 {[T, Hq]} on {dev}")
    return t.data_ptr()


def _cache(k: torch.Tensor, v: torch.Tensor, pages: torch.Tensor, dev: torch.device) -> LatentKvCache:
    if k.dim() != 4 or v.shape != k.shape:
        raise ValueError("k_cache and v_cache must be [pages, page rows, kv heads, D], of one shape")
    if k.dtype not in _DTYPE or v.dtype != k.dtype:
        raise TypeError("the cache must be f16 or bf16, keys and values alike")
    if k.device != dev or v.device != dev or pages.device != dev:
        raise ValueError(f"the cache and its page table must be on {dev}")
    if pages.dtype != torch.int32 or pages.dim() != 2 or (pages.stride(1) != 1 and pages.shape[1] > 1):
        raise ValueError("pages must be int32 [sequences, max_pages], its rows adjacent")
    n, page, heads, D = k.shape
    ks, vs = k.stride(), v.stride()
    if (ks[3] != 1 or vs[3] != 1) and D > 1:
        raise ValueError("the last dimension of k_cache and v_cache must be adjacent")
    B, most = pages.shape
    # A size of one makes its stride meaningless to torch, and so to the library.
    return LatentKvCache(k.data_ptr(), v.data_ptr(), pages.data_ptr(), n, page, B, most,
                         pages.stride(0) if B > 1 else most, ks[0] if n > 1 else 0, ks[1] if page > 1 else 0,
                         ks[2] if heads > 1 else 0, vs[0] if n > 1 else 0, vs[1] if page > 1 else 0,
                         vs[2] if heads > 1 else 0)


def _first(t: torch.Tensor, name: str) -> torch.device:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dtype not in _DTYPE:
        raise TypeError(f"{name} must be f16 or bf16")
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("attention here has no backward pass: call it under torch.no_grad()")
    return t.device


def _here(t: torch.Tensor, stream: Optional[torch.cuda.Stream]):
    """The context a call has to enter first: its stream's or its tensors' device's; None when both are current."""
    if stream is not None:
        return torch.cuda.stream(stream)
    if t.is_cuda and t.device.index != torch.cuda.current_device():
        return torch.cuda.device(t.device)
    return None


def _stream(dev: torch.device) -> int:
    return torch.cuda.current_stream(dev).cuda_stream


def _scale(scale: Optional[float], D: int) -> float:
    s = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not 0.0 < s < math.inf:
        raise ValueError("scale must be positive and finite")
    return s


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
    ctx = _here(k, stream)
    if ctx is not None:
        with ctx:
            return kv_append(k, v, k_cache, v_cache, pages, positions, seqs, q, rope, interleaved, q_out)
    dev = _first(k, "k")
    dt = k.dtype
    cache = _cache(k_cache, v_cache, pages, dev)
    k, v = _heads(k, "k", dt, dev), _heads(v, "v", dt, dev)
    T, Hkv, D = k.shape
    if k_cache.dtype != dt or k_cache.shape[2:] != (Hkv, D) or v.shape != k.shape:
        raise ValueError(f"k {list(k.shape)}, v {list(v.shape)} and the cache {list(k_cache.shape)} {k_cache.dtype} do not fit")
    if seqs is None and T > cache.n_seq:
        raise ValueError("more tokens than sequences: give seqs")
    positions = _ints(positions, "positions", (T,), dev)
    if seqs is not None:
        seqs = _ints(seqs, "seqs", (T,), dev)
    rows = rot = rp = 0
    if rope is not None:
        if rope.dtype != torch.float32 or rope.dim() != 3 or rope.shape[1] != 2 or rope.device != dev:
            raise ValueError(f"rope must be f32 [positions, 2, rot / 2] on {dev}")
        if not rope.is_contiguous() or rope.data_ptr() % 16:
            rope = rope.contiguous().clone()
        rows, rot, rp = rope.shape[0], 2 * rope.shape[2], rope.data_ptr()
        if not 0 < rot <= D:
            raise ValueError(f"rope turns {rot} dimensions of {D}")
    Hq = 0
    qp = op = (0, 0, 0)
    if q is not None:
        q = _heads(q, "q", dt, dev)
        if q.shape[0] != T or q.shape[2] != D:
            raise ValueError(f"q {list(q.shape)} does not fit k {list(k.shape)}")
        q_out = _out(q_out, q, "q_out")
        Hq = q.shape[1]
        qp, op = (q.data_ptr(), *q.stride()[:2]), (q_out.data_ptr(), *q_out.stride()[:2])
    elif q_out is not None:
        raise ValueError("q_out without q")
    if T == 0:
        return q_out
    a = LatentKvAppendArgs(cache, qp[0], op[0], k.data_ptr(), v.data_ptr(), qp[1], qp[2], op[1], op[2], *k.stride()[:2],
                           *v.stride()[:2], positions.data_ptr(), 0 if seqs is None else seqs.data_ptr(), rp, rows, rot, T,
                           Hq, Hkv, D, _DTYPE[dt], int(interleaved))
    check(lib.latent_kv_append(ctypes.byref(a), _stream(dev)), "latent_kv_append")
    return q_out


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
    ctx = _here(q, stream)
    if ctx is not None:
        with ctx:
            return attend_decode(q, k_cache, v_cache, pages, lengths, scale, out, lse, workspace)
    dev = _first(q, "q")
    cache = _cache(k_cache, v_cache, pages, dev)
    q = _heads(q, "q", k_cache.dtype, dev)
    B, Hq, D = q.shape
    Hkv = k_cache.shape[2]
    if B != cache.n_seq or D != k_cache.shape[3] or not Hkv or Hq % Hkv:
        raise ValueError(f"q {list(q.shape)} does not fit the cache {list(k_cache.shape)} of {cache.n_seq} sequences")
    lengths = _ints(lengths, "lengths", (B,), dev)
    out = _out(out, q, "out")
    lp = _lse(lse, B, Hq, dev)
    if B == 0 or Hq == 0:
        return out
    a = LatentAttnDecodeArgs(cache, q.data_ptr(), out.data_ptr(), lp, lengths.data_ptr(), *q.stride()[:2], *out.stride()[:2],
                             Hq, Hkv, D, _DTYPE[q.dtype], _scale(scale, D))
    if workspace is None:
        n = ctypes.c_size_t()
        check(lib.latent_attn_decode_workspace_size(ctypes.byref(a), ctypes.byref(n)), "latent_attn_decode_workspace_size")
        workspace = torch.empty(n.value, dtype=torch.uint8, device=dev)
    elif workspace.device != dev or not workspace.is_contiguous():
        raise ValueError(f"workspace must be contiguous and on {dev}")
    a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    check(lib.latent_attn_decode(ctypes.byref(a), _stream(dev)), "latent_attn_decode")
    return out


def attend_decode_workspace_size(n_seq: int, n_head: int, n_kv_head: int, head_dim: int, max_pages: int, page_size: int) -> int:
    """Workspace bytes of attend_decode for these sizes."""
    c = LatentKvCache(n_pages=1, page_size=page_size, n_seq=n_seq, max_pages=max_pages, pages_stride=max_pages)
    a = LatentAttnDecodeArgs(cache=c, n_head=n_head, n_kv_head=n_kv_head, head_dim=head_dim, dtype=_lib.LATENT_BF16, scale=1.0)
    n = ctypes.c_size_t()
    check(lib.latent_attn_decode_workspace_size(ctypes.byref(a), ctypes.byref(n)), "latent_attn_decode_workspace_size")
    return int(n.value)


def _prompt(q, starts, cache, Hkv, kv, lengths, causal, scale, out, lse, dev) -> torch.Tensor:
    T, Hq, D = q.shape
    B = cache.n_seq
    if not Hkv or Hq % Hkv:
        raise ValueError(f"{Hq} heads are no multiple of {Hkv} key and value heads")
    starts = _ints(starts, "starts", (B + 1,), dev)
    out = _out(out, q, "out")
    lp = _lse(lse, T, Hq, dev)
    if T == 0 or Hq == 0 or B == 0:
        return out
    k, v, k_starts = kv
    a = LatentAttnPromptArgs(cache, q.data_ptr(), out.data_ptr(), lp, 0 if k is None else k.data_ptr(),
                             0 if k is None else v.data_ptr(), starts.data_ptr(), 0 if k is None else k_starts.data_ptr(),
                             0 if lengths is None else lengths.data_ptr(), *q.stride()[:2], *out.stride()[:2],
                             *((0, 0) if k is None else k.stride()[:2]), *((0, 0) if k is None else v.stride()[:2]), T,
                             0 if k is None else k.shape[0], Hq, Hkv, D, _DTYPE[q.dtype], int(causal), _scale(scale, D))
    check(lib.latent_attn_prompt(ctypes.byref(a), _stream(dev)), "latent_attn_prompt")
    return out


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
    stream: Optional[torch.cuda.Stream] = None,
) -> torch.Tensor:
    """Whole prompts, packed: sequence b is rows starts[b] .. starts[b + 1] - 1 (int32 [B + 1], ascending) of
    q [T, heads, D] and of k, v [Tk, kv heads, D] (rows k_starts[b] .. where k_starts is given).

    Causal with the ends aligned: with n queries and m keys, query i sees keys
    j <= i + m - n.  Rows of out and lse (f32 [T, heads]) that belong to no
    sequence are not written; a row that sees no key is zeros, lse -inf.
    """
    ctx = _here(q, stream)
    if ctx is not None:
        with ctx:
            return attend_prompt(q, k, v, starts, k_starts, causal, scale, out, lse)
    dev = _first(q, "q")
    q, k, v = _heads(q, "q", q.dtype, dev), _heads(k, "k", q.dtype, dev), _heads(v, "v", q.dtype, dev)
    if v.shape != k.shape or k.shape[2] != q.shape[2]:
        raise ValueError(f"q {list(q.shape)}, k {list(k.shape)} and v {list(v.shape)} do not fit")
    if k_starts is None:
        if k.shape[0] != q.shape[0]:
            raise ValueError("k has other rows than q: give k_starts")
        k_starts = starts
    if starts.dim() != 1 or starts.shape[0] == 0:
        raise ValueError("starts must be int32 [sequences + 1]")
    B = starts.shape[0] - 1
    k_starts = _ints(k_starts, "k_starts", (B + 1,), dev)
    cache = LatentKvCache(n_seq=B, page_size=1)
    return _prompt(q, starts, cache, k.shape[1], (k, v, k_starts), None, causal, scale, out, lse, dev)


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
    stream: Optional[torch.cuda.Stream] = None,
) -> torch.Tensor:
    """attend_prompt with the keys and values of sequence b in the cache: its first lengths[b] (int32 [B])
    positions, the new tokens' own (appended before the call) the last of them."""
    ctx = _here(q, stream)
    if ctx is not None:
        with ctx:
            return attend_prompt_paged(q, k_cache, v_cache, pages, lengths, starts, causal, scale, out, lse)
    dev = _first(q, "q")
    cache = _cache(k_cache, v_cache, pages, dev)
    q = _heads(q, "q", k_cache.dtype, dev)
    if q.shape[2] != k_cache.shape[3]:
        raise ValueError(f"q {list(q.shape)} does not fit the cache {list(k_cache.shape)}")
    lengths = _ints(lengths, "lengths", (cache.n_seq,), dev)
    return _prompt(q, starts, cache, k_cache.shape[2], (None, None, None), lengths, causal, scale, out, lse, dev)
