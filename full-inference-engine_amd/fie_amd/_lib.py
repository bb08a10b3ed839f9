"""ctypes binding of the C ABI in include/fie_sampler.h, include/fie_ops.h and include/fie_decode.h.

The shared library is built in-tree by ``fie_amd.build`` into ``fie_amd/_native``.
There is no fallback: if the library cannot be loaded, every entry point raises.
"""

from __future__ import annotations

import ctypes
import os

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "_native", "libfie_sampler.so")

FIE_OK = 0
FIE_E_ARG, FIE_E_WORKSPACE, FIE_E_LAUNCH = -1, -2, -3
FIE_F32, FIE_F16, FIE_BF16, FIE_I8 = 0, 1, 2, 3
FIE_FLAG_GREEDY, FIE_FLAG_PENALTY, FIE_FLAG_NO_DRAW = 1, 2, 4
FIE_ROW_EXACT_PATH = 1
FIE_ROW_UNCOUNTED_IDS = 2
FIE_STAGE_PREP, FIE_STAGE_SCAN, FIE_STAGE_FINISH, FIE_STAGE_DEEP = 0, 1, 2, 3
LP_COLS = 20
TILE = 8192
MAX_VOCAB = 64 * TILE
MAX_DRAFTS = 255
VERIFY_DRAWS_VOCAB = 63488

_vp = ctypes.c_void_p


class SamplerArgs(ctypes.Structure):
    """Mirror of ``fie_sampler_args``."""

    _fields_ = [
        ("logits", _vp), ("dtype", ctypes.c_int32), ("rows", ctypes.c_int32),
        ("vocab", ctypes.c_int32), ("lp_cols", ctypes.c_int32), ("row_stride", ctypes.c_int64),
        ("scale", _vp), ("top_k", _vp), ("top_p", _vp), ("min_p", _vp), ("flags", _vp),
        ("logprobs", _vp), ("uniform", _vp),
        ("apply_penalties", ctypes.c_int32), ("max_row_hist", ctypes.c_int32),
        ("repetition", _vp), ("presence", _vp), ("frequency", _vp),
        ("hist_offsets", _vp), ("hist_ids", _vp), ("hist_invalid", _vp),
        ("tokens", _vp), ("status", _vp), ("tk_key", _vp), ("cut_comp", _vp),
        ("row_max", _vp), ("kept_mass", _vp), ("row_mass", _vp), ("chosen_logprob", _vp),
        ("top_ids", _vp), ("top_logprobs", _vp), ("rng", _vp), ("hist_ends", _vp),
    ]


class VerifyArgs(ctypes.Structure):
    """Mirror of ``fie_verify_args``."""

    _fields_ = [
        ("requests", ctypes.c_int32), ("max_drafts", ctypes.c_int32), ("draft_offsets", _vp), ("draft_ids", _vp),
        ("draft_probs", _vp), ("draft_dtype", ctypes.c_int32), ("draws", ctypes.c_int32),
        ("draft_stride", ctypes.c_int64), ("tokens", _vp), ("accepted", _vp), ("target_probs", _vp),
    ]


# ``fie_norm_args`` and ``fie_int8_args`` as struct formats, native sizes and alignment (filling
# a ctypes structure of as many fields takes four times as long): pointers and sizes as P and q,
# a trailing 0 quad pads to the structure's alignment.
NORM_ARGS = "@10P6q9i3f0q"
INT8_ARGS = "@6P4q4iPN0q"
BEAM_ARGS = "@15PqPNd8i18i0q"
ADAPTER_ARGS = "@10PN3q12i0q"
ADAPTER_PLAN_ARGS = "@2P2i0q"
PAGES_ARGS, GROUP_ARGS = "@PPN4i6P2i", "P3q4i"          # the head, and eight groups
STATES_ARGS, STATE_ARGS = "@P2i", "2P4q"        # the head, and as many states as there are


class Workspace(ctypes.Structure):
    """Mirror of ``fie_workspace``."""

    _fields_ = [("ptr", _vp), ("bytes", ctypes.c_size_t), ("max_rows", ctypes.c_int32),
                ("vocab", ctypes.c_int32)]


# Every symbol include/fie_sampler.h declares.
EXPORTS = (
    "fie_sampler_workspace_size", "fie_sampler_sample", "fie_sampler_stage",
    "fie_sampler_argmax", "fie_sampler_kept", "fie_sampler_cexp", "fie_sampler_last_error",
    "fie_sampler_sample_noalloc", "fie_sampler_uniforms", "fie_sampler_history_write",
    "fie_sampler_lmhead_sample", "fie_sampler_lmhead_stage", "fie_sampler_verify",
)
# Every symbol include/fie_ops.h declares.
OPS_EXPORTS = ("fie_block_norm", "fie_int8_linear", "fie_int8_workspace_size")
# Every symbol include/fie_decode.h declares.
DECODE_EXPORTS = ("fie_beam_workspace_size", "fie_beam_step", "fie_reorder_states", "fie_pages_state_ints",
                  "fie_pages_scratch_bytes", "fie_pages_step", "fie_pages_compact", "fie_pages_copy", "fie_adapter_plan_ints",
                  "fie_adapter_plan", "fie_adapter_workspace_size", "fie_adapter_linear")
SCRATCH_BYTES = 64 << 20

_lib = None


class NativeError(RuntimeError):
    pass


def load():
    """Load the HIP library (import torch first so both share one HIP runtime)."""
    global _lib
    if _lib is not None:
        return _lib
    import torch  # noqa: F401  -- the HIP runtime must come from torch's process image

    if not os.path.exists(LIB_PATH):
        raise NativeError(
            f"the HIP sampler library is not built ({LIB_PATH}); run fie_amd.build.build()")
    lib = ctypes.CDLL(LIB_PATH)
    bind(lib)
    _lib = lib
    return lib


def bind(lib) -> None:
    """Declare argument and result types of every exported function."""
    lib.fie_sampler_workspace_size.restype = ctypes.c_size_t
    lib.fie_sampler_workspace_size.argtypes = [ctypes.c_int32, ctypes.c_int32]
    lib.fie_sampler_sample.argtypes = [ctypes.POINTER(SamplerArgs), ctypes.POINTER(Workspace), _vp]
    lib.fie_sampler_stage.argtypes = [
        ctypes.POINTER(SamplerArgs), ctypes.POINTER(Workspace), ctypes.c_int32, _vp]
    lib.fie_sampler_argmax.argtypes = [
        _vp, ctypes.c_int32, ctypes.c_int32, ctypes.c_int32, ctypes.c_int64, _vp,
        ctypes.POINTER(Workspace), _vp]
    lib.fie_sampler_kept.argtypes = [
        ctypes.POINTER(SamplerArgs), _vp, _vp, ctypes.POINTER(Workspace), _vp]
    lib.fie_sampler_cexp.argtypes = [_vp, _vp, ctypes.c_int64, _vp]
    lib.fie_sampler_sample_noalloc.argtypes = [ctypes.POINTER(SamplerArgs), _vp]
    lib.fie_sampler_uniforms.argtypes = [_vp, _vp, ctypes.c_int32, _vp]
    lib.fie_sampler_history_write.argtypes = [_vp, _vp, _vp, ctypes.c_int64, _vp]
    for name in ("fie_sampler_lmhead_sample", "fie_sampler_lmhead_stage"):
        getattr(lib, name).argtypes = [ctypes.POINTER(SamplerArgs), _vp, _vp, ctypes.c_int32,
                                       ctypes.POINTER(Workspace), _vp]
    lib.fie_sampler_verify.argtypes = [ctypes.POINTER(SamplerArgs), ctypes.POINTER(VerifyArgs),
                                       ctypes.POINTER(Workspace), _vp]
    lib.fie_sampler_last_error.restype = ctypes.c_char_p
    lib.fie_block_norm.argtypes = [ctypes.c_char_p, _vp]
    lib.fie_int8_linear.argtypes = [ctypes.c_char_p, _vp]
    for name in ("fie_beam_step", "fie_reorder_states", "fie_pages_step", "fie_pages_compact", "fie_pages_copy",
                 "fie_adapter_plan", "fie_adapter_linear"):
        getattr(lib, name).argtypes = [ctypes.c_char_p, _vp]
    for name in EXPORTS + OPS_EXPORTS + DECODE_EXPORTS:
        if name not in ("fie_sampler_workspace_size", "fie_sampler_last_error"):
            getattr(lib, name).restype = ctypes.c_int
    lib.fie_beam_workspace_size.argtypes = [ctypes.c_char_p]
    lib.fie_beam_workspace_size.restype = ctypes.c_size_t
    lib.fie_adapter_plan_ints.argtypes = [ctypes.c_int32] * 2
    lib.fie_adapter_workspace_size.argtypes = [ctypes.c_char_p]
    lib.fie_adapter_plan_ints.restype = lib.fie_adapter_workspace_size.restype = ctypes.c_size_t
    lib.fie_pages_state_ints.argtypes = [ctypes.c_int32] * 3
    lib.fie_pages_scratch_bytes.argtypes = [ctypes.c_int32] * 2
    lib.fie_pages_state_ints.restype = lib.fie_pages_scratch_bytes.restype = ctypes.c_size_t
    lib.fie_int8_workspace_size.argtypes = [ctypes.c_char_p]
    lib.fie_int8_workspace_size.restype = ctypes.c_size_t


def launcher(name: str):
    """``run(index, *args)``: the library's function ``name`` on device ``index`` and its current
    stream (the interpreter's own calls for both take a tenth of the time of torch.cuda's
    wrappers)."""
    import torch

    fn = getattr(load(), name)
    get, stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream

    def run(index: int, *args) -> None:
        if get() == index:
            rc = fn(*args, stream(index))
        else:
            with torch.cuda.device(index):
                rc = fn(*args, stream(index))
        if rc != FIE_OK:
            check(rc, name)

    return run


def check(rc: int, what: str) -> None:
    if rc != FIE_OK:
        msg = _lib.fie_sampler_last_error().decode() if _lib is not None else ""
        raise NativeError(f"{what} failed ({rc}): {msg}")
