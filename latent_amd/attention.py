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
import functools
import math
import struct
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import LatentAttnDecodeArgs, LatentAttnPromptArgs, LatentKvAppendArgs, check, lib

try:  # the current stream's handle without a Stream object: 0.1 instead of 1.9 us of a call
    from torch._C import _cuda_getCurrentRawStream as _stream
except ImportError:
    def _stream(device: int) -> int:
        return torch.cuda.current_stream(device).cuda_stream

_DTYPE = {torch.float16: _lib.LATENT_F16, torch.bfloat16: _lib.LATENT_BF16}


def _packer(args):
    """The argument struct of ctypes class `args` from its values in field order, as bytes (0.3 us; a nested ctypes
    structure takes 1.5)."""
    codes = {ctypes.c_void_p: "q", ctypes.c_int64: "q", ctypes.c_size_t: "q", ctypes.c_int32: "i", ctypes.c_float: "f"}

    def fields(c):
        return "".join(fields(t) if issubclass(t, ctypes.Structure) else codes[t] for _, t in c._fields_)

    s = struct.Struct("@" + fields(args) + "0q")
    assert s.size == ctypes.sizeof(args)
    return s.pack


def _entry(name: str):
    """The library's function on packed arguments."""
    f = lib[name]
    f.restype, f.argtypes = ctypes.c_int, [ctypes.c_char_p, ctypes.c_void_p]
    return f


_append_args, _append = _packer(LatentKvAppendArgs), _entry("latent_kv_append")
_decode_args, _decode = _packer(LatentAttnDecodeArgs), _entry("latent_attn_decode")
_decode_size = _entry("latent_attn_decode_workspace_size")
_prompt_args, _prompt_call = _packer(LatentAttnPromptArgs), _entry("latent_attn_prompt")
_prompt_size = _entry("latent_attn_prompt_workspace_size")


def rope_table(n_positions: int, rot_dim: int, base: float = 10000.0, device="cuda") -> torch.Tensor:
    """cos and sin of position p times base^(-2i / rot_dim), f32 [n_positions, 2, rot_dim / 2]
    (angles in 64 bits: in 32 a far position's angle is off by more than the table's rounding)."""
    if n_positions < 0 or rot_dim <= 0 or rot_dim % 2:
        raise ValueError("rot_dim must be even and positive")
    i = torch.arange(0, rot_dim, 2, dtype=torch.float64, device=device)
    angle = torch.arange(n_positions, dtype=torch.float64, device=device)[:, None] * base ** (-i / rot_dim)
    return torch.stack((angle.cos(), angle.sin()), 1).float().contiguous()


def _no_grad():
    raise RuntimeError("attention here has no backward pass: call it under torch.no_grad()")


def _heads(t: torch.Tensor, name: str, dt: torch.dtype, dev: int):
    """[T, heads, D] as the kernels read it (a copy where strides or base do not fit), its base, strides and shape."""
    shape = t.shape
    if len(shape) != 3:
        raise ValueError(f"{name} must be [tokens, heads, D]")
    if t.dtype is not dt:
        raise TypeError(f"{name} must be {dt}, as the queries and the cache are")
    if t.get_device() != dev:
        raise ValueError(f"{name} must be on cuda:{dev}")
    if t.requires_grad and torch.is_grad_enabled():
        _no_grad()
    st, sh, sd = t.stride()
    p = t.data_ptr()
    if (sd != 1 and shape[2] > 1) or (st | sh) & 7 or p & 15 or st >= _FAR:
        t = t.clone(memory_format=torch.contiguous_format)
        st, sh, sd = t.stride()
        p = t.data_ptr()
    return t, p, st, sh, shape


# Tokens further apart than this (elements) are copied together: the kernels step over a tile of them in 32 bits.
_FAR = 1 << 22


def _ints(t: torch.Tensor, name: str, n: int, dev: int) -> torch.Tensor:
    if t.dtype is not torch.int32 or t.dim() != 1 or t.numel() != n or t.get_device() != dev:
        raise ValueError(f"{name} must be int32 [{n}] on cuda:{dev}")
    return t if t.is_contiguous() else t.contiguous()


def _out(t: Optional[torch.Tensor], like: torch.Tensor, name: str):
    """The output, its base and strides."""
    if t is None:
        t = torch.empty_like(like, memory_format=torch.contiguous_format)
        return t, t.data_ptr(), *t.stride()[:2]
    if t.shape != like.shape or t.dtype is not like.dtype or t.get_device() != like.get_device():
        raise ValueError(f"{name} must be {like.dtype} {list(like.shape)} on {like.device}")
    if t.requires_grad and torch.is_grad_enabled():
        _no_grad()
    st, sh, sd = t.stride()
    if (sd != 1 and t.shape[2] > 1) or (st | sh) & 7 or t.data_ptr() & 15:
        raise ValueError(f"{name} must have adjacent D, strides that are multiples of 8 and a 16-byte aligned base")
    return t, t.data_ptr(), st, sh


def _lse(t: Optional[torch.Tensor], T: int, Hq: int, dev: int) -> int:
    if t is None:
        return 0
    if t.dtype is not torch.float32 or tuple(t.shape) != (T, Hq) or t.get_device() != dev or not t.is_contiguous():
        raise ValueError(f"lse must be contiguous f32 {[T, Hq]} on cuda:{dev}")
    return t.data_ptr()


def _cache(k: torch.Tensor, v: torch.Tensor, pages: torch.Tensor, dev: int):
    """The fields of a LatentKvCache, and the cache's shape and type."""
    shape, dt = k.shape, k.dtype
    if len(shape) != 4 or v.shape != shape:
        raise ValueError("k_cache and v_cache must be [pages, page rows, kv heads, D], of one shape")
    if dt not in _DTYPE or v.dtype is not dt:
        raise TypeError("the cache must be f16 or bf16, keys and values alike")
    if (k.requires_grad or v.requires_grad) and torch.is_grad_enabled():
        _no_grad()
    if k.get_device() != dev or v.get_device() != dev or pages.get_device() != dev:
        raise ValueError(f"the cache and its page table must be on cuda:{dev}")
    B_most = pages.shape
    if pages.dtype is not torch.int32 or len(B_most) != 2:
        raise ValueError("pages must be int32 [sequences, max_pages]")
    B, most = B_most
    ps, one = pages.stride()
    n, page, heads, D = shape
    k0, k1, k2, k3 = k.stride()
    v0, v1, v2, v3 = v.stride()
    if ((k3 != 1 or v3 != 1) and D > 1) or (one != 1 and most > 1):
        raise ValueError("the last dimensions of k_cache, v_cache and pages must be adjacent")
    # A size of one makes its stride meaningless to torch, and so to the library.
    if B < 2 or n < 2 or page < 2 or heads < 2:
        ps = ps if B > 1 else most
        k0, v0 = (k0, v0) if n > 1 else (0, 0)
        k1, v1 = (k1, v1) if page > 1 else (0, 0)
        k2, v2 = (k2, v2) if heads > 1 else (0, 0)
    return (k.data_ptr(), v.data_ptr(), pages.data_ptr(), n, page, B, most, ps, k0, k1, k2, v0, v1, v2), shape, dt


def _first(t: torch.Tensor, name: str) -> int:
    """The device of a call's first tensor."""
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dtype not in _DTYPE:
        raise TypeError(f"{name} must be f16 or bf16")
    return t.get_device()


def _here(t: torch.Tensor, stream: Optional[torch.cuda.Stream]):
    """The context a call has to enter first: its stream's or its tensors' device's; None when both are current."""
    if stream is not None:
        return torch.cuda.stream(stream)
    if t.is_cuda and t.get_device() != torch.cuda.current_device():
        return torch.cuda.device(t.device)
    return None


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
    cache, (_, _, cHkv, cD), cdt = _cache(k_cache, v_cache, pages, dev)
    k, kp, kt, kh, kshape = _heads(k, "k", dt, dev)
    v, vp, vt, vh, vshape = _heads(v, "v", dt, dev)
    T, Hkv, D = kshape
    if cdt is not dt or cHkv != Hkv or cD != D or vshape != kshape:
        raise ValueError(f"k {list(k.shape)}, v {list(v.shape)} and the cache {list(k_cache.shape)} {k_cache.dtype} do not fit")
    sp = rows = rot = rp = 0
    if seqs is not None:
        seqs = _ints(seqs, "seqs", T, dev)
        sp = seqs.data_ptr()
    elif T > cache[5]:
        raise ValueError("more tokens than sequences: give seqs")
    positions = _ints(positions, "positions", T, dev)
    if rope is not None:
        if rope.dtype is not torch.float32 or rope.dim() != 3 or rope.shape[1] != 2 or rope.get_device() != dev:
            raise ValueError(f"rope must be f32 [positions, 2, rot / 2] on cuda:{dev}")
        rp = rope.data_ptr()
        if not rope.is_contiguous() or rp & 15:
            rope = rope.clone(memory_format=torch.contiguous_format)
            rp = rope.data_ptr()
        rows, _, rot = rope.shape
        rot *= 2
        if not 0 < rot <= D:
            raise ValueError(f"rope turns {rot} dimensions of {D}")
    qp = qt = qh = op = ot = oh = Hq = 0
    if q is not None:
        q, qp, qt, qh, (Tq, Hq, Dq) = _heads(q, "q", dt, dev)
        if Tq != T or Dq != D:
            raise ValueError(f"q {list(q.shape)} does not fit k {list(k.shape)}")
        q_out, op, ot, oh = _out(q_out, q, "q_out")
    elif q_out is not None:
        raise ValueError("q_out without q")
    if T == 0:
        return q_out
    a = _append_args(*cache, qp, op, kp, vp, qt, qh, ot, oh, kt, kh, vt, vh, positions.data_ptr(), sp, rp, rows, rot, T, Hq,
                     Hkv, D, _DTYPE[dt], 1 if interleaved else 0)
    st = _append(a, _stream(dev))
    if st:
        check(st, "latent_kv_append")
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
    cache, (_, _, Hkv, cD), dt = _cache(k_cache, v_cache, pages, dev)
    q, qp, qt, qh, (B, Hq, D) = _heads(q, "q", dt, dev)
    if B != cache[5] or D != cD or not Hkv or Hq % Hkv:
        raise ValueError(f"q {list(q.shape)} does not fit the cache {list(k_cache.shape)} of {cache[5]} sequences")
    lengths = _ints(lengths, "lengths", B, dev)
    out, op, ot, oh = _out(out, q, "out")
    lp = _lse(lse, B, Hq, dev)
    if B == 0 or Hq == 0:
        return out
    a = (*cache, qp, op, lp, lengths.data_ptr(), qt, qh, ot, oh, Hq, Hkv, D, _DTYPE[dt], _scale(scale, D))
    if workspace is None:
        n = _decode_need(*cache[4:7], Hq, Hkv, D)
        if n:
            workspace = torch.empty(n, dtype=torch.uint8, device=q.device)
    elif workspace.get_device() != dev or not workspace.is_contiguous():
        raise ValueError(f"workspace must be contiguous and on cuda:{dev}")
    else:
        n = workspace.numel() * workspace.element_size()
    st = _decode(_decode_args(*a, workspace.data_ptr() if n else 0, n), _stream(dev))
    if st:
        check(st, "latent_attn_decode")
    return out


@functools.lru_cache(maxsize=256)
def _decode_need(page_size: int, n_seq: int, max_pages: int, n_head: int, n_kv_head: int, head_dim: int) -> int:
    cache = (0, 0, 0, 1, page_size, n_seq, max_pages, max_pages, 0, 0, 0, 0, 0, 0)
    n = ctypes.c_size_t()
    a = _decode_args(*cache, *(0,) * 8, n_head, n_kv_head, head_dim, _lib.LATENT_BF16, 1.0, 0, 0)
    check(_decode_size(a, ctypes.addressof(n)), "latent_attn_decode_workspace_size")
    return int(n.value)


def attend_decode_workspace_size(n_seq: int, n_head: int, n_kv_head: int, head_dim: int, max_pages: int, page_size: int) -> int:
    """Workspace bytes of attend_decode for these sizes."""
    return _decode_need(page_size, n_seq, max_pages, n_head, n_kv_head, head_dim)


def _prompt(q, starts, cache, Hkv, keys, k_starts, lengths, n_keys, causal, scale, out, lse, workspace, dev) -> torch.Tensor:
    """keys: base and strides of k and v, (k, v, k token, k head, v token, v head), zeros for the cache's."""
    q, qp, qt, qh, (T, Hq, D) = q
    B = cache[5]
    if not Hkv or Hq % Hkv:
        raise ValueError(f"{Hq} heads are no multiple of {Hkv} key and value heads")
    starts = _ints(starts, "starts", B + 1, dev)
    out, op, ot, oh = _out(out, q, "out")
    lp = _lse(lse, T, Hq, dev)
    if T == 0 or Hq == 0 or B == 0:
        return out
    if workspace is None:
        need = _prompt_need(T, B, n_keys, cache[6] * cache[4], Hq, Hkv, D)
        if need:
            workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    elif workspace.get_device() != dev or not workspace.is_contiguous():
        raise ValueError(f"workspace must be contiguous and on cuda:{dev}")
    else:
        need = workspace.numel() * workspace.element_size()
    a = _prompt_args(*cache, qp, op, lp, keys[0], keys[1], starts.data_ptr(), 0 if k_starts is None else k_starts.data_ptr(),
                     0 if lengths is None else lengths.data_ptr(), qt, qh, ot, oh, *keys[2:], T, n_keys, Hq, Hkv, D,
                     _DTYPE[q.dtype], 1 if causal else 0, _scale(scale, D), workspace.data_ptr() if need else 0, need)
    st = _prompt_call(a, _stream(dev))
    if st:
        check(st, "latent_attn_prompt")
    return out


@functools.lru_cache(maxsize=1024)
def _prompt_need(n_tokens: int, n_seq: int, n_keys: int, cached: int, n_head: int, n_kv_head: int, head_dim: int) -> int:
    cache = (0, 0, 0, 1, 1, n_seq, cached, cached, 0, 0, 0, 0, 0, 0)
    n = ctypes.c_size_t()
    a = _prompt_args(*cache, *(0,) * 16, n_tokens, n_keys, n_head, n_kv_head, head_dim, _lib.LATENT_BF16, 1, 1.0, 0, 0)
    check(_prompt_size(a, ctypes.addressof(n)), "latent_attn_prompt_workspace_size")
    return int(n.value)


def attend_prompt_workspace_size(n_tokens: int, n_seq: int, n_head: int, n_kv_head: int, head_dim: int, n_keys: int = 0,
                                 max_pages: int = 0, page_size: int = 1) -> int:
    """Workspace bytes of attend_prompt (n_keys rows of keys) or attend_prompt_paged for these sizes; 0: it takes none."""
    return _prompt_need(n_tokens, n_seq, n_keys, 0 if n_keys else max_pages * page_size, n_head, n_kv_head, head_dim)


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
    ctx = _here(q, stream)
    if ctx is not None:
        with ctx:
            return attend_prompt(q, k, v, starts, k_starts, causal, scale, out, lse, workspace)
    dev = _first(q, "q")
    dt = q.dtype
    q = _heads(q, "q", dt, dev)
    k, kp, kt, kh, (Tk, Hkv, D) = _heads(k, "k", dt, dev)
    v, vp, vt, vh, vshape = _heads(v, "v", dt, dev)
    if vshape != k.shape or D != q[4][2]:
        raise ValueError(f"q {list(q[4])}, k {list(k.shape)} and v {list(vshape)} do not fit")
    if starts.dim() != 1 or starts.shape[0] == 0:
        raise ValueError("starts must be int32 [sequences + 1]")
    B = starts.shape[0] - 1
    if k_starts is None:
        if Tk != q[4][0]:
            raise ValueError("k has other rows than q: give k_starts")
        k_starts = starts
    k_starts = _ints(k_starts, "k_starts", B + 1, dev)
    if Tk == 0:  # a tensor without rows has no base
        kp = vp = q[1]
    cache = (0, 0, 0, 0, 1, B, 0, 0, 0, 0, 0, 0, 0, 0)
    return _prompt(q, starts, cache, Hkv, (kp, vp, kt, kh, vt, vh), k_starts, None, Tk, causal, scale, out, lse, workspace, dev)


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
    positions, the new tokens' own (appended before the call) the last of them."""
    ctx = _here(q, stream)
    if ctx is not None:
        with ctx:
            return attend_prompt_paged(q, k_cache, v_cache, pages, lengths, starts, causal, scale, out, lse, workspace)
    dev = _first(q, "q")
    cache, (_, _, Hkv, cD), dt = _cache(k_cache, v_cache, pages, dev)
    q = _heads(q, "q", dt, dev)
    if q[4][2] != cD:
        raise ValueError(f"q {list(q[4])} does not fit the cache {list(k_cache.shape)}")
    lengths = _ints(lengths, "lengths", cache[5], dev)
    return _prompt(q, starts, cache, Hkv, (0,) * 6, None, lengths, 0, causal, scale, out, lse, workspace, dev)


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
        qkv = (x.to(self.w_qkv.dtype) @ self.w_qkv).view(x.shape[0], -1, self.head_dim)
        H, K = self.n_head, self.n_kv_head
        q = qkv[:, :H]
        return kv_append(qkv[:, H:H + K], qkv[:, H + K:], self.k_cache, self.v_cache, pages, positions, seqs=seqs,
                         q=q, rope=self.rope, interleaved=self.interleaved, q_out=q)

    def _project(self, a: torch.Tensor) -> torch.Tensor:
        return a.view(a.shape[0], -1) @ self.w_o

    def decode(self, x: torch.Tensor, pages: torch.Tensor, positions: torch.Tensor, lengths: torch.Tensor,
               workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
        """One new token a sequence: x [B, d] at positions [B]; lengths [B] count it.  Returns [B, d] in the weights' type."""
        q = self._append(x, pages, positions, None)
        return self._project(attend_decode(q, self.k_cache, self.v_cache, pages, lengths, scale=self.scale, workspace=workspace))

    def prompt(self, x: torch.Tensor, pages: torch.Tensor, positions: torch.Tensor, seqs: torch.Tensor, starts: torch.Tensor,
               lengths: torch.Tensor) -> torch.Tensor:
        """New tokens of several sequences, packed: x [T, d], token t of sequence seqs[t] (row of pages) at positions[t],
        sequence b's being rows starts[b] .. starts[b + 1] - 1 and the last of its lengths[b].  Rows of no sequence
        (padding, at negative positions) give zeros."""
        q = self._append(x, pages, positions, seqs)
        out = torch.zeros_like(q, memory_format=torch.contiguous_format)
        return self._project(attend_prompt_paged(q, self.k_cache, self.v_cache, pages, lengths, starts, scale=self.scale, out=out))
