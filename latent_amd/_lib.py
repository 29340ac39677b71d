"""ctypes binding of liblatent_hip.so (include/latent_ffn.h).

The library is loaded after `import torch`, so it shares torch's HIP runtime:
`tensor.data_ptr()` and `torch.cuda.current_stream().cuda_stream` are passed
straight through.  There is no fallback: if the library is missing, importing
this module raises.
"""

from __future__ import annotations

import ctypes
import os
from pathlib import Path

import torch  # noqa: F401  (must precede the CDLL load; see module docstring)

# LATENT_HIP_LIB points at another build of the same library (e.g. a debug build).
LIB_PATH = Path(os.environ.get("LATENT_HIP_LIB", Path(__file__).resolve().parent / "liblatent_hip.so"))

LATENT_OK = 0
LATENT_E_INVALID = -1
LATENT_E_UNSUPPORTED = -2
LATENT_E_WORKSPACE = -3
LATENT_E_HIP = -4
LATENT_E_TIMEOUT = -5

LATENT_F32 = 0
LATENT_F16 = 1
LATENT_BF16 = 2

LATENT_OUT_REDUCED = 0
LATENT_OUT_PER_SLOT = 1

LATENT_LAYOUT_ROWS = 0
LATENT_LAYOUT_TILES = 1

# Factor indices of latent_tiles_repack, in the operand order.
LATENT_GATE_A, LATENT_GATE_B, LATENT_UP_A, LATENT_UP_B, LATENT_DOWN_A, LATENT_DOWN_B = range(6)

EXPORTED = (
    "latent_version",
    "latent_status_string",
    "latent_moe_workspace_size",
    "latent_moe_ffn_forward",
    "latent_moe_ffn_forward_noalloc",
    "latent_moe_path",
    "latent_stream_launch",
    "latent_moe_check",
    "latent_unpack",
    "latent_pack_nf4",
    "latent_pack_int8",
    "latent_route_workspace_size",
    "latent_route",
    "latent_expert_workspace_size",
    "latent_expert_forward",
    "latent_tiles_supported",
    "latent_tiles_repack",
    "latent_kv_append",
    "latent_attn_decode_workspace_size",
    "latent_attn_decode",
    "latent_attn_prompt_workspace_size",
    "latent_attn_prompt",
    "latent_kv_append_q8",
    "latent_kv_read",
    "latent_attn_decode_q8_workspace_size",
    "latent_attn_decode_q8",
    "latent_attn_prompt_q8",
    "latent_attn_decode_shared_workspace_size",
    "latent_attn_decode_shared",
    "latent_residual_norm",
)

LATENT_NOALLOC_SCRATCH_BYTES = 64 << 20
LATENT_NOALLOC_CONTROL_BYTES = 256 << 10

LATENT_Q_NF4 = 0
LATENT_Q_INT8 = 1

LATENT_DROP_NONE = 0
LATENT_DROP_BELOW = 1
LATENT_DROP_INCLUSIVE = 2


class LatentFactor(ctypes.Structure):
    _fields_ = [
        ("codes", ctypes.c_void_p),
        ("scales", ctypes.c_void_p),
        ("int8_bitmap", ctypes.c_void_p),
        ("int8_row_offset", ctypes.c_void_p),
        ("int8_data", ctypes.c_void_p),
        ("rows", ctypes.c_int64),
        ("cols", ctypes.c_int64),
    ]


class LatentMoeArgs(ctypes.Structure):
    _fields_ = [
        ("x", ctypes.c_void_p),
        ("x_dtype", ctypes.c_int32),
        ("ids", ctypes.c_void_p),
        ("weights", ctypes.c_void_p),
        ("weights_dtype", ctypes.c_int32),
        ("gate_a", LatentFactor),
        ("gate_b", LatentFactor),
        ("up_a", LatentFactor),
        ("up_b", LatentFactor),
        ("down_a", LatentFactor),
        ("down_b", LatentFactor),
        ("ranks", ctypes.c_void_p),
        ("n_tokens", ctypes.c_int64),
        ("n_embd", ctypes.c_int64),
        ("n_ff", ctypes.c_int64),
        ("n_expert", ctypes.c_int64),
        ("n_expert_used", ctypes.c_int64),
        ("max_rank", ctypes.c_int64),
        ("weight_before_down", ctypes.c_int32),
        ("out_mode", ctypes.c_int32),
        ("out", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_size_t),
        ("layout", ctypes.c_int32),
    ]


class LatentRouteArgs(ctypes.Structure):
    _fields_ = [
        ("x", ctypes.c_void_p),
        ("x_dtype", ctypes.c_int32),
        ("router", ctypes.c_void_p),
        ("router_dtype", ctypes.c_int32),
        ("logits_in", ctypes.c_void_p),
        ("logits_out", ctypes.c_void_p),
        ("ids", ctypes.c_void_p),
        ("weights", ctypes.c_void_p),
        ("n_tokens", ctypes.c_int64),
        ("n_embd", ctypes.c_int64),
        ("n_expert", ctypes.c_int64),
        ("n_expert_used", ctypes.c_int64),
        ("drop_rule", ctypes.c_int32),
        ("drop_param", ctypes.c_float),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_size_t),
    ]


class LatentFlatFactor(ctypes.Structure):
    _fields_ = [
        ("data", ctypes.c_void_p),
        ("scales", ctypes.c_void_p),
        ("kind", ctypes.c_int32),
        ("group_size", ctypes.c_int32),
        ("rows", ctypes.c_int64),
        ("cols", ctypes.c_int64),
    ]


class LatentExpertArgs(ctypes.Structure):
    _fields_ = [
        ("x", ctypes.c_void_p),
        ("gate_a", LatentFlatFactor),
        ("gate_b", LatentFlatFactor),
        ("up_a", LatentFlatFactor),
        ("up_b", LatentFlatFactor),
        ("down_a", LatentFlatFactor),
        ("down_b", LatentFlatFactor),
        ("n_tokens", ctypes.c_int64),
        ("weight", ctypes.c_float),
        ("weight_before_down", ctypes.c_int32),
        ("out", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_size_t),
    ]


LATENT_ROPE_HALF = 0
LATENT_ROPE_INTERLEAVED = 1


class LatentKvCache(ctypes.Structure):
    _fields_ = [
        ("k", ctypes.c_void_p),
        ("v", ctypes.c_void_p),
        ("pages", ctypes.c_void_p),
        *[(n, ctypes.c_int64) for n in (
            "n_pages", "page_size", "n_seq", "max_pages", "pages_stride", "k_page_stride", "k_row_stride",
            "k_head_stride", "v_page_stride", "v_row_stride", "v_head_stride")],
    ]


class LatentKvAppendArgs(ctypes.Structure):
    _fields_ = [
        ("cache", LatentKvCache),
        *[(n, ctypes.c_void_p) for n in ("q", "q_out", "k", "v")],
        *[(n, ctypes.c_int64) for n in (
            "q_token_stride", "q_head_stride", "q_out_token_stride", "q_out_head_stride", "k_token_stride",
            "k_head_stride", "v_token_stride", "v_head_stride")],
        *[(n, ctypes.c_void_p) for n in ("positions", "seqs", "rope")],
        *[(n, ctypes.c_int64) for n in ("rope_rows", "rot_dim", "n_tokens", "n_head", "n_kv_head", "head_dim")],
        ("dtype", ctypes.c_int32),
        ("rope_kind", ctypes.c_int32),
    ]


class LatentAttnDecodeArgs(ctypes.Structure):
    _fields_ = [
        ("cache", LatentKvCache),
        *[(n, ctypes.c_void_p) for n in ("q", "out", "lse", "lengths")],
        *[(n, ctypes.c_int64) for n in (
            "q_token_stride", "q_head_stride", "out_token_stride", "out_head_stride", "n_head", "n_kv_head",
            "head_dim")],
        ("dtype", ctypes.c_int32),
        ("scale", ctypes.c_float),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_size_t),
    ]


class LatentAttnPromptArgs(ctypes.Structure):
    _fields_ = [
        ("cache", LatentKvCache),
        *[(n, ctypes.c_void_p) for n in ("q", "out", "lse", "k", "v", "starts", "k_starts", "lengths")],
        *[(n, ctypes.c_int64) for n in (
            "q_token_stride", "q_head_stride", "out_token_stride", "out_head_stride", "k_token_stride",
            "k_head_stride", "v_token_stride", "v_head_stride", "n_tokens", "n_keys", "n_head", "n_kv_head",
            "head_dim")],
        ("dtype", ctypes.c_int32),
        ("causal", ctypes.c_int32),
        ("scale", ctypes.c_float),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_size_t),
    ]


LATENT_CODE_INT8 = 0
LATENT_CODE_E4M3 = 1


class LatentKvScales(ctypes.Structure):
    _fields_ = [
        ("k", ctypes.c_void_p),
        ("v", ctypes.c_void_p),
        *[(n, ctypes.c_int64) for n in ("k_page_stride", "k_head_stride", "v_page_stride", "v_head_stride")],
        ("code", ctypes.c_int32),
    ]


class LatentKvReadArgs(ctypes.Structure):
    _fields_ = [
        ("cache", LatentKvCache),
        *[(n, ctypes.c_void_p) for n in ("k", "v")],
        *[(n, ctypes.c_int64) for n in ("k_token_stride", "k_head_stride", "v_token_stride", "v_head_stride")],
        *[(n, ctypes.c_void_p) for n in ("positions", "seqs")],
        *[(n, ctypes.c_int64) for n in ("n_tokens", "n_kv_head", "head_dim")],
        ("dtype", ctypes.c_int32),
    ]


class LatentAttnSharedArgs(ctypes.Structure):
    _fields_ = [
        ("decode", LatentAttnDecodeArgs),
        ("scales", ctypes.POINTER(LatentKvScales)),
        ("prefix", ctypes.c_void_p),
        ("n_prefix", ctypes.c_int64),
    ]


LATENT_NORM_NONE = 0
LATENT_NORM_RMS = 1
LATENT_NORM_LAYER = 2


class LatentNorm(ctypes.Structure):
    _fields_ = [
        ("kind", ctypes.c_int32),
        ("eps", ctypes.c_float),
        ("weight", ctypes.c_void_p),
        ("bias", ctypes.c_void_p),
        ("dtype", ctypes.c_int32),
    ]


class LatentResidualNormArgs(ctypes.Structure):
    _fields_ = [
        *[(n, ctypes.c_void_p) for n in ("x", "y", "gate", "x_out", "n_out")],
        *[(n, ctypes.c_int64) for n in ("x_stride", "y_stride", "gate_stride", "x_out_stride", "n_out_stride", "n_tokens", "n_embd")],
        *[(n, ctypes.c_int32) for n in ("x_dtype", "y_dtype", "gate_dtype", "n_dtype")],
        ("scale", ctypes.c_float),
        ("post", LatentNorm),
        ("pre", LatentNorm),
    ]


class LatentError(RuntimeError):
    def __init__(self, status: int, what: str):
        super().__init__(f"{what}: {status_string(status)} ({status})")
        self.status = status


def _load() -> ctypes.CDLL:
    if not LIB_PATH.exists():
        raise ImportError(
            f"{LIB_PATH} is missing: build it with `python latent_amd/build.py` "
            "(there is no CPU fallback)"
        )
    lib = ctypes.CDLL(str(LIB_PATH))
    lib.latent_version.restype = ctypes.c_int
    lib.latent_version.argtypes = []
    lib.latent_status_string.restype = ctypes.c_char_p
    lib.latent_status_string.argtypes = [ctypes.c_int]
    lib.latent_moe_workspace_size.restype = ctypes.c_int
    lib.latent_moe_workspace_size.argtypes = [ctypes.POINTER(LatentMoeArgs), ctypes.POINTER(ctypes.c_size_t)]
    lib.latent_moe_ffn_forward.restype = ctypes.c_int
    lib.latent_moe_ffn_forward.argtypes = [ctypes.POINTER(LatentMoeArgs), ctypes.c_void_p]
    lib.latent_moe_check.restype = ctypes.c_int
    lib.latent_moe_check.argtypes = [ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]
    lib.latent_moe_ffn_forward_noalloc.restype = ctypes.c_int
    lib.latent_moe_ffn_forward_noalloc.argtypes = [ctypes.POINTER(LatentMoeArgs), ctypes.c_void_p]
    lib.latent_moe_path.restype = ctypes.c_int
    lib.latent_moe_path.argtypes = [ctypes.POINTER(LatentMoeArgs)]
    lib.latent_stream_launch.restype = ctypes.c_int
    lib.latent_stream_launch.argtypes = [ctypes.POINTER(LatentMoeArgs)]
    lib.latent_unpack.restype = ctypes.c_int
    lib.latent_unpack.argtypes = [ctypes.POINTER(LatentFactor), ctypes.c_int64, ctypes.c_void_p, ctypes.c_void_p]
    lib.latent_pack_nf4.restype = ctypes.c_int
    lib.latent_pack_nf4.argtypes = [
        ctypes.c_void_p, ctypes.c_int64, ctypes.c_int64, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p,
    ]
    lib.latent_pack_int8.restype = ctypes.c_int
    lib.latent_pack_int8.argtypes = [ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p]
    lib.latent_route_workspace_size.restype = ctypes.c_int
    lib.latent_route_workspace_size.argtypes = [ctypes.POINTER(LatentRouteArgs), ctypes.POINTER(ctypes.c_size_t)]
    lib.latent_route.restype = ctypes.c_int
    lib.latent_route.argtypes = [ctypes.POINTER(LatentRouteArgs), ctypes.c_void_p]
    lib.latent_expert_workspace_size.restype = ctypes.c_int
    lib.latent_expert_workspace_size.argtypes = [ctypes.POINTER(LatentExpertArgs), ctypes.POINTER(ctypes.c_size_t)]
    lib.latent_expert_forward.restype = ctypes.c_int
    lib.latent_expert_forward.argtypes = [ctypes.POINTER(LatentExpertArgs), ctypes.c_void_p]
    lib.latent_tiles_supported.restype = ctypes.c_int
    lib.latent_tiles_supported.argtypes = [ctypes.POINTER(LatentMoeArgs)]
    lib.latent_tiles_repack.restype = ctypes.c_int
    lib.latent_tiles_repack.argtypes = [
        ctypes.c_int32, ctypes.POINTER(LatentFactor), ctypes.POINTER(LatentFactor), ctypes.c_int64, ctypes.c_int32,
        ctypes.c_void_p,
    ]
    lib.latent_kv_append.restype = ctypes.c_int
    lib.latent_kv_append.argtypes = [ctypes.POINTER(LatentKvAppendArgs), ctypes.c_void_p]
    lib.latent_attn_decode_workspace_size.restype = ctypes.c_int
    lib.latent_attn_decode_workspace_size.argtypes = [
        ctypes.POINTER(LatentAttnDecodeArgs), ctypes.POINTER(ctypes.c_size_t),
    ]
    lib.latent_attn_decode.restype = ctypes.c_int
    lib.latent_attn_decode.argtypes = [ctypes.POINTER(LatentAttnDecodeArgs), ctypes.c_void_p]
    lib.latent_attn_prompt_workspace_size.restype = ctypes.c_int
    lib.latent_attn_prompt_workspace_size.argtypes = [
        ctypes.POINTER(LatentAttnPromptArgs), ctypes.POINTER(ctypes.c_size_t),
    ]
    lib.latent_attn_prompt.restype = ctypes.c_int
    lib.latent_attn_prompt.argtypes = [ctypes.POINTER(LatentAttnPromptArgs), ctypes.c_void_p]
    size = ctypes.POINTER(ctypes.c_size_t)
    for name, args in (
        ("kv_append_q8", (ctypes.POINTER(LatentKvAppendArgs), ctypes.POINTER(LatentKvScales), ctypes.c_void_p)),
        ("kv_read", (ctypes.POINTER(LatentKvReadArgs), ctypes.POINTER(LatentKvScales), ctypes.c_void_p)),
        ("attn_decode_q8_workspace_size", (ctypes.POINTER(LatentAttnDecodeArgs), size)),
        ("attn_decode_q8", (ctypes.POINTER(LatentAttnDecodeArgs), ctypes.POINTER(LatentKvScales), ctypes.c_void_p)),
        ("attn_prompt_q8", (ctypes.POINTER(LatentAttnPromptArgs), ctypes.POINTER(LatentKvScales), ctypes.c_void_p)),
        ("attn_decode_shared_workspace_size", (ctypes.POINTER(LatentAttnSharedArgs), size)),
        ("attn_decode_shared", (ctypes.POINTER(LatentAttnSharedArgs), ctypes.c_void_p)),
        ("residual_norm", (ctypes.POINTER(LatentResidualNormArgs), ctypes.c_void_p)),
    ):
        f = lib[f"latent_{name}"]
        setattr(lib, f"latent_{name}", f)
        f.restype, f.argtypes = ctypes.c_int, list(args)
    return lib


lib = _load()


def status_string(status: int) -> str:
    return lib.latent_status_string(int(status)).decode()


def check(status: int, what: str) -> None:
    if status != LATENT_OK:
        raise LatentError(status, what)
