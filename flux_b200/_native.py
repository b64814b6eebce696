"""ctypes binding of ``libfluxb200.so`` (the C ABI declared in ``include/flux_b200.h``).

The library is the only compute path.  If it has not been built, every entry
point raises :class:`NativeLibraryUnavailable` -- there is no CPU fallback.
"""

from __future__ import annotations

import ctypes
import hashlib
import mmap
import os
from pathlib import Path

LIBRARY_PATH = Path(__file__).resolve().parent / "_lib" / "libfluxb200.so"
LAYERS = 30

FX_OK = 0
FX_ERR_INVALID = 1
FX_ERR_CUDA = 2
FX_ERR_EXHAUSTED = 3
FX_ERR_STATE = 4
FX_ERR_DEVICE = 5

STATE_POSITION = 0
STATE_CACHE_LENGTH = 1
STATE_GENERATION_STEP = 2

_p = ctypes.c_void_p
_i64 = ctypes.c_int64
_i32 = ctypes.c_int32
_f32 = ctypes.c_float
_st = ctypes.c_int32


class NativeLibraryUnavailable(RuntimeError):
    """``libfluxb200.so`` is missing or failed to load."""


class ModelDesc(ctypes.Structure):
    """``fx_model_desc``."""

    _fields_ = [
        ("device", _i32),
        ("vocab", _i64),
        ("capacity", _i64),
        ("epsilon", _f32),
        ("embedding", _p),
        ("final_norm", _p),
        ("lm_head", _p),
        ("rope_cos", _p),
        ("rope_sin", _p),
        ("input_norm", _p * LAYERS),
        ("packed_qkv", _p * LAYERS),
        ("o_proj", _p * LAYERS),
        ("post_norm", _p * LAYERS),
        ("gate_up", _p * LAYERS),
        ("down", _p * LAYERS),
        ("attention_scale", _f32 * LAYERS),
    ]


class DecodeBuffers(ctypes.Structure):
    """``fx_decode_buffers``."""

    _fields_ = [
        ("input_token", _p),
        ("logits", _p),
        ("generated_tokens", _p),
        ("generation_step", _p),
        ("key_cache", _p),
        ("value_cache", _p),
        ("position", _p),
        ("cache_length", _p),
        ("workspace", _p),
        ("workspace_bytes", _i64),
        ("hidden_a", _p),
        ("hidden_b", _p),
        ("final_norm_output", _p),
        ("attention_workspace", _p),
        ("stable_buffer_bytes", _i64),
        ("timeline", _p),
        ("timeline_ctas", _i64),
        ("timeline_events", _i64),
    ]


class DecodeInfo(ctypes.Structure):
    """``fx_decode_info``."""

    _fields_ = [
        ("capacity", _i64),
        ("vocab", _i64),
        ("start_position", _i64),
        ("replay_count", _i64),
        ("kernels_per_step", _i64),
    ]


class PrefillBuffers(ctypes.Structure):
    """``fx_prefill_buffers``."""

    _fields_ = [
        ("prefill_logits", _p),
        ("workspace", _p),
        ("workspace_bytes", _i64),
        ("attention_output", _p),
        ("final_hidden", _p),
        ("initial_token", _p),
    ]


class BatchBuffers(ctypes.Structure):
    """``fx_batch_buffers``."""

    _fields_ = [
        ("tokens", _p),
        ("positions", _p),
        ("logits", _p),
        ("generated", _p),
        ("step", _p),
        ("key_cache", _p),
        ("value_cache", _p),
        ("batch", _i64),
        ("capacity", _i64),
        ("generated_capacity", _i64),
        ("kernels_per_step", _i64),
    ]


class Pages(ctypes.Structure):
    """``fx_pages``."""

    _fields_ = [
        ("keys", _p),
        ("values", _p),
        ("dtype", _i32),
        ("layers", _i64),
        ("pages", _i64),
        ("kv_heads", _i64),
        ("page_size", _i64),
        ("head_dim", _i64),
        ("key_strides", _i64 * 4),
        ("value_strides", _i64 * 4),
    ]


# name -> (restype, argtypes)
SIGNATURES: dict[str, tuple] = {
    "fx_last_error": (ctypes.c_char_p, []),
    "fx_version": (ctypes.c_char_p, []),
    "fx_rmsnorm_f32": (_st, [_p, _p, _p, _i64, _i64, _f32, _p]),
    "fx_residual_rmsnorm_f32": (_st, [_p, _p, _p, _p, _p, _i64, _i64, _f32, _p]),
    "fx_packed_swiglu_f32": (_st, [_p, _p, _i64, _i64, _p]),
    "fx_softmax_f32": (_st, [_p, _p, _i64, _i64, _p]),
    "fx_attention_score_softmax_f32": (_st, [_p, _p, _p, _p, _p, _f32, _p, _p]),
    "fx_rope_f32": (_st, [_p, _p, _p, _p, _p, _p, _p, _p, _p, _p, _i64, _i64, _i64, _i64, _i64, _i64, _p]),
    "fx_packed_qkv_rope_cache_f32": (_st, [_p, _p, _p, _p, _p, _p, _p, _p, _p, _p, _i64, _p, _p, _p, _p]),
    "fx_gqa_decode_attention_workspace_floats": (_i64, [_i64, _i64, _i64, _i64]),
    "fx_gqa_decode_attention_f32": (_st, [_p, _p, _p, _p, _p, _p, _p, _p, _p, _p, _p, _p, _i64, _f32,
                                          _i64, _i64, _i64, _i64, _i64, _p]),
    "fx_gqa_decode_attention_static_scratch_floats": (_i64, []),
    "fx_gqa_decode_attention_static_scratch_f32": (_st, [_p, _p, _p, _p, _p, _p, _p, _p, _p, _p, _p, _f32,
                                                         _i64, _i64, _i64, _i64, _i64, _p]),
    "fx_packed_gate_up_swiglu_f32": (_st, [_p, _p, _p, _i64, _i64, _p]),
    "fx_linear_f32": (_st, [_p, _p, _p, _i64, _i64, _i64, _p]),
    "fx_tf32_split_f32": (_st, [_p, _p, _p, _i64, _p]),
    "fx_linear_3xtf32_f32": (_st, [_p, _p, _p, _p, _p, _i64, _i64, _i64, _p, _p]),
    "fx_greedy_argmax_f32": (_st, [_p, _i64, _p, _p]),
    "fx_greedy_argmax_update_f32": (_st, [_p, _i64, _p, _p, _i64, _p, _p, _p, _p]),
    "fx_paged_qkv_rope_cache": (_st, [_p, _i32, _i64, _i64, _i64, _p, _i64, _p, _i64, _i64, ctypes.POINTER(Pages), _p,
                                      _i64, _i64, _i64, _p, _p, _p, _p]),
    "fx_paged_gqa_decode_attention_workspace_floats": (_i64, [_i64, _i64, _i64]),
    "fx_paged_gqa_decode_attention": (_st, [_p, _i32, _p, _i64, _i64, ctypes.POINTER(Pages), _p, _i64, _i64, _p, _f32,
                                            _p, _p, _i64, _p]),
    "fx_cache_pages_copy": (_st, [ctypes.POINTER(Pages), _p, _p, _i64, _p]),
    "fx_cache_sequences_reserve": (_st, [_p, _i64, _i64, _i64, _p, _p, _i64, _i64, _p, _p, _i64, _p, _p, _p]),
    "fx_cache_sequences_fork": (_st, [ctypes.POINTER(Pages), _p, _i64, _i64, _i64, _p, _p, _p, _p, _i64, _p, _p, _p]),
    "fx_cache_sequences_free": (_st, [_p, _i64, _i64, _i64, _p, _p, _i64, _p, _i64, _p]),
    "fx_cache_pages_compact": (_st, [ctypes.POINTER(Pages), _p, _i64, _i64, _i64, _p, _p, _p, _p]),
    "fx_logits_process": (_st, [_p, _i32, _i64, _i64, _i64, _p, _i64, _i64, _p, _p, _p, _p, _i64, _p, _i64, _p, _i64,
                                _p]),
    "fx_decode_create": (_st, [ctypes.POINTER(ModelDesc), _p, _p, _p, _i64, _i64, _p, ctypes.POINTER(_p)]),
    "fx_decode_replay": (_st, [_p, _p, _p]),
    "fx_decode_replay_host": (_st, [_p, _p, _p, _p]),
    "fx_decode_generate": (_st, [_p, _i64, _p]),
    "fx_decode_reset": (_st, [_p, _p, _p, _p, _i64, _i64, _p]),
    "fx_decode_inject_failure": (_st, [_p, ctypes.c_int32]),
    "fx_decode_set_eos": (_st, [_p, _i64]),
    "fx_decode_install_prefill": (_st, [_p, _p, _i64, _p]),
    "fx_decode_wait": (_st, [_p, _p]),
    "fx_decode_get_buffers": (_st, [_p, ctypes.POINTER(DecodeBuffers)]),
    "fx_decode_read_state": (_st, [_p, _i32, ctypes.POINTER(_i64)]),
    "fx_decode_get_info": (_st, [_p, ctypes.POINTER(DecodeInfo)]),
    "fx_decode_destroy": (None, [_p]),
    "fx_batch_create": (_st, [ctypes.POINTER(ModelDesc), _i64, _i64, _p, ctypes.POINTER(_p)]),
    "fx_batch_load": (_st, [_p, _i64, _p, _p, _p, _i64, _i64, _p]),
    "fx_batch_step": (_st, [_p, _i64, _p]),
    "fx_batch_wait": (_st, [_p, _p]),
    "fx_batch_check": (_st, [_p]),
    "fx_batch_get_buffers": (_st, [_p, ctypes.POINTER(BatchBuffers)]),
    "fx_batch_destroy": (None, [_p]),
    "fx_prefill_create": (_st, [ctypes.POINTER(ModelDesc), _p, _i64, _p, ctypes.POINTER(_p)]),
    "fx_prefill_run": (_st, [_p, _p, _p]),
    "fx_prefill_decode": (_p, [_p]),
    "fx_prefill_get_buffers": (_st, [_p, ctypes.POINTER(PrefillBuffers)]),
    "fx_prefill_prompt_length": (_i64, [_p]),
    "fx_prefill_destroy": (None, [_p]),
}

_LIB: ctypes.CDLL | None = None
_LOAD_ERROR: Exception | None = None


def _missing(library: Path, names) -> str | None:
    """The first of the names that the library's file does not hold, if any.  The
    file is looked through before it is loaded: a loaded library stays, and
    would be found again in the place of one rebuilt at the same path."""
    with open(library, "rb") as file:
        if os.fstat(file.fileno()).st_size == 0:
            return next(iter(names))
        with mmap.mmap(file.fileno(), 0, access=mmap.ACCESS_READ) as data:
            return next((name for name in names if data.find(name.encode() + b"\0") < 0), None)


def load(path: str | os.PathLike | None = None) -> ctypes.CDLL:
    """Load (once) and return the library with every signature declared."""
    global _LIB, _LOAD_ERROR
    if _LIB is not None:
        return _LIB
    target = Path(path) if path is not None else LIBRARY_PATH
    if not target.exists():
        _LOAD_ERROR = NativeLibraryUnavailable(
            f"flux_b200 native library is not built ({target} is missing); "
            "run `python -m flux_b200.build`")
        raise _LOAD_ERROR
    missing = _missing(target, SIGNATURES)
    if missing is not None:
        _LOAD_ERROR = NativeLibraryUnavailable(
            f"{target} is an older build, without {missing}; run `python -m flux_b200.build`")
        raise _LOAD_ERROR
    try:
        lib = ctypes.CDLL(str(target))
    except OSError as error:
        _LOAD_ERROR = NativeLibraryUnavailable(f"failed to load {target}: {error}")
        raise _LOAD_ERROR from error
    for name, (restype, argtypes) in SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype = restype
        fn.argtypes = argtypes
    _LIB = lib
    _LOAD_ERROR = None
    return lib


TORCH_CLASSES_PATH = LIBRARY_PATH.with_name("libfluxb200_torch.so")
TORCH_ENTRIES = ["paged_gqa_decode_attention", "logits_process"]  # operators it has to register
torch_classes_loaded = False


def load_torch_classes() -> bool:
    """Register ``torch.classes.flux.NativeSmolLM2Decode`` / ``NativeSmolLM2Prefill``
    and the serving operators of ``torch.ops.flux`` (``libfluxb200_torch.so``,
    the reference's custom-class surface and the paged-cache and logits
    operators over this library); False when that library is not built, older
    than the package or does not load, until it does: only success is remembered, so a process may build
    the library and go on.  The C library loads first so both share one copy of
    it."""
    global torch_classes_loaded
    if not torch_classes_loaded and TORCH_CLASSES_PATH.exists():
        try:
            load()
            if _missing(TORCH_CLASSES_PATH, TORCH_ENTRIES) is not None:
                return False  # an older build
            import torch
            torch.classes.load_library(str(TORCH_CLASSES_PATH))
            torch_classes_loaded = True
        except (OSError, RuntimeError, NativeLibraryUnavailable):
            pass
    return torch_classes_loaded


# Written by the build: the digest of the sources that the libraries were built from.
SOURCES_PATH = LIBRARY_PATH.with_name("sources.sha256")


def sources_digest() -> str:
    package = LIBRARY_PATH.parents[1]
    files = [*package.glob("csrc/*"), *package.parent.glob("include/*.h")]
    h = hashlib.sha256()
    for path in sorted(p for p in files if p.suffix in (".cu", ".cuh", ".cpp", ".h")):
        h.update(f"{path.name} {path.stat().st_size}\n".encode())
        h.update(path.read_bytes())
    return h.hexdigest()


def load_current_torch_classes() -> bool:
    """:func:`load_torch_classes` for the import of the package, where no one
    has asked for the library yet: one built from other sources is left alone,
    since a process that goes on to rebuild it could not load the new one."""
    try:
        current = SOURCES_PATH.read_text() == sources_digest()
    except OSError:
        return False
    return current and load_torch_classes()


def is_available() -> bool:
    try:
        load()
    except NativeLibraryUnavailable:
        return False
    return True


def load_error() -> Exception | None:
    try:
        load()
    except NativeLibraryUnavailable:
        pass
    return _LOAD_ERROR


class NativeError(RuntimeError):
    """A non-zero ``fx_status``; ``status`` keeps the code."""

    def __init__(self, status: int, message: str):
        super().__init__(message)
        self.status = status


def check(status: int) -> None:
    if status != FX_OK:
        message = load().fx_last_error().decode("utf-8", "replace")
        raise NativeError(status, message or f"flux_b200 call failed with status {status}")


def int64_array(values) -> ctypes.Array:
    values = [int(v) for v in values]
    return (_i64 * len(values))(*values)


def pointer_array(values) -> ctypes.Array:
    values = [int(v) for v in values]
    return (_p * len(values))(*values)
