"""Block norms: the end of one block and the norm in front of the next, in one pass.

    z = gate * post_norm(x)
    r = residual + scale * z
    y = norm(r)

with the norm over the last dimension (RMS or layer), everything in fp32 between the loads and
the stores; ``y`` optionally in 8-bit integers with a scale for each token, as
``fie_amd.linear.int8_linear`` takes it (a token with a NaN has the scale NaN, and its products are
NaN).
"""

from __future__ import annotations

import struct
from typing import NamedTuple

import torch

from . import _lib
from ._lib import FIE_BF16, FIE_F16, FIE_F32, FIE_I8

_DTYPES = {torch.float32: FIE_F32, torch.float16: FIE_F16, torch.bfloat16: FIE_BF16}
_KINDS = {"rms": 0, "layer": 1, "none": 2}
_pack = struct.Struct(_lib.NORM_ARGS).pack
_run = None             # the library's entry, loaded with the first call
MAX_WIDTH = 65536
MAX_K = 131071          # of a quantisation alone: as wide as the 8-bit product takes its rows


class BlockNorm(NamedTuple):
    residual: torch.Tensor | None       # residual + scale * z, in the residual's type
    y: torch.Tensor                     # its norm: x's type, or int8
    scale: torch.Tensor | None          # float32 [tokens] with int8


def _launch(index: int, args: bytes) -> None:
    global _run
    if _run is None:
        _run = _lib.launcher("fie_block_norm")
    _run(index, args)


def _rows(t: torch.Tensor, width: int) -> torch.Tensor:
    """[tokens, width] with unit element stride (a copy where the view has none)."""
    if t.ndim != 2:
        t = t.reshape(-1, width)
    return t if t.stride(1) == 1 or width == 1 else t.contiguous()


def block_norm(residual: torch.Tensor, x: torch.Tensor | None = None, weight: torch.Tensor | None = None, *,
               bias: torch.Tensor | None = None, post_weight: torch.Tensor | None = None,
               post_bias: torch.Tensor | None = None, post_norm: bool | None = None,
               gate: torch.Tensor | None = None, scale: float = 1.0, eps: float = 1e-6, kind: str = "rms",
               weight_offset: float = 0.0, quantize: bool = False,
               out_dtype: torch.dtype | None = None, inplace: bool = False) -> BlockNorm:
    """``norm(residual + scale * gate * post_norm(x))`` and the residual in front of it.

    ``residual`` and ``x`` [..., width] share a shape; the residual is in x's type or float32.
    Without ``x`` the norm is of the residual alone (no new residual; ``out_dtype`` is y's type,
    the residual's by default).  ``post_norm`` defaults to whether ``post_weight`` is given.
    ``gate``: [width], x's shape, or x's shape with a last dimension of 1.  ``kind``: "rms",
    "layer" or "none" (y is r itself).  ``weight_offset`` is added to both weights.  Parameters
    are in x's type or float32 (weights and biases all in one).  ``inplace`` writes the new
    residual over the old.  Runs on the current stream; nothing waits for it."""
    shape = residual.shape
    width = shape[-1] if shape else 0
    if not 1 <= width <= MAX_WIDTH:
        raise ValueError(f"residual must be [..., width] with width in [1, {MAX_WIDTH}]")
    r_dtype = _DTYPES.get(residual.dtype)
    if r_dtype is None:
        raise ValueError("residual must be float32, float16 or bfloat16")
    norm = _KINDS.get(kind)
    if norm is None:
        raise ValueError("kind must be 'rms', 'layer' or 'none'")
    if x is None:
        dtype = out_dtype if out_dtype is not None else residual.dtype
        if gate is not None or post_norm or post_weight is not None or post_bias is not None or inplace:
            raise ValueError("gate, post norm and inplace need x")
    else:
        dtype = x.dtype
        if x.shape != shape:
            raise ValueError("x and residual must have one shape")
        if residual.dtype != dtype and residual.dtype != torch.float32:
            raise ValueError("residual is in x's type or float32")
        if out_dtype is not None and out_dtype != dtype:
            raise ValueError("out_dtype is x's type")
    x_dtype = _DTYPES.get(dtype)
    if x_dtype is None:
        raise ValueError("x and out_dtype must be float32, float16 or bfloat16")
    index = residual.get_device()
    if index < 0:
        raise ValueError("block_norm runs on a HIP device")
    post = post_norm if post_norm is not None else post_weight is not None
    # parameter vectors: all in x's type, or all in float32
    vectors, v_dtype = [0, 0, 0, 0], None
    for i, t in enumerate((weight, bias, post_weight, post_bias)):
        if t is None:
            continue
        if t.ndim != 1 or t.shape[0] != width or not t.is_contiguous():
            raise ValueError(f"weights and biases must be contiguous vectors of {width}")
        if v_dtype is None:
            v_dtype = t.dtype
            if v_dtype != dtype and v_dtype != torch.float32:
                raise ValueError(f"weights and biases must be in {dtype} or float32")
        if t.dtype != v_dtype or t.get_device() != index:
            raise ValueError("weights and biases must share one type, on the residual's device")
        if norm == 2:
            raise ValueError("kind 'none' takes no norm parameters")
        if i >= 2 and not post:
            raise ValueError("post parameters without post_norm")
        vectors[i] = t.data_ptr()
    if norm == 2 and post:
        raise ValueError("kind 'none' takes no norm parameters")
    flat = len(shape) == 2
    res = residual if flat and (residual.stride(1) == 1 or width == 1) else _rows(residual, width)
    tokens, r_stride = res.shape[0], res.stride(0)
    device = residual.device
    new = xs = gp = None
    xp = x_stride = n_ptr = n_stride = g_ptr = g_stride = g_step = g_f32 = 0
    if x is not None:
        xs = x if flat and (x.stride(1) == 1 or width == 1) else _rows(x, width)
        xp, x_stride = xs.data_ptr(), xs.stride(0)
        if x.get_device() != index:
            raise ValueError("x must be on the residual's device")
        if inplace:
            if res.data_ptr() != residual.data_ptr() or (tokens > 1 and r_stride < width):
                raise ValueError("inplace needs a residual with unit element stride and rows that do not overlap")
            new, n_stride = res, r_stride
        else:
            new = torch.empty_like(res) if r_stride == width else torch.empty((tokens, width), dtype=residual.dtype, device=device)
            n_stride = width
        n_ptr = new.data_ptr()
        if gate is not None:
            if gate.get_device() != index or (gate.dtype != dtype and gate.dtype != torch.float32):
                raise ValueError(f"gate must be in {dtype} or float32, on the residual's device")
            if gate.shape == (width,):
                gp, g_stride, g_step = gate.contiguous(), 0, 1
            elif gate.shape == shape:
                gp = _rows(gate, width)
                g_stride, g_step = gp.stride(0), 1
            elif gate.shape == (*shape[:-1], 1):
                gp = gate.reshape(-1)
                g_stride, g_step = gp.stride(0), 0
            else:
                raise ValueError("gate must be [width], x's shape, or x's shape with a last dimension of 1")
            g_ptr, g_f32 = gp.data_ptr(), gate.dtype == torch.float32
    like = res if xs is None else xs
    if not quantize and like.dtype == dtype and like.stride(0) == width:
        y = torch.empty_like(like)
    else:
        y = torch.empty((tokens, width), dtype=torch.int8 if quantize else dtype, device=device)
    y_scale = torch.empty(tokens, dtype=torch.float32, device=device) if quantize else None
    if tokens:
        _launch(index, _pack(xp, res.data_ptr(), n_ptr, y.data_ptr(), y_scale.data_ptr() if quantize else 0, *vectors, g_ptr,
                             tokens, x_stride, r_stride, n_stride, width, g_stride, g_step, width, x_dtype, r_dtype,
                             FIE_I8 if quantize else x_dtype, v_dtype == torch.float32, g_f32, norm, post, scale, eps,
                             weight_offset))
    if not flat:
        y = y.view(shape)
        if new is not None and not inplace:
            new = new.view(shape)
    return BlockNorm(residual if inplace else new, y, y_scale)


def quantized(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [..., width] in int8 [tokens, width], and its rows' scales: what ``block_norm`` of kind "none"
    gives with ``quantize``, without its other arguments' checks, and up to MAX_K wide."""
    shape = x.shape
    width = shape[-1] if shape else 0
    if not 1 <= width <= MAX_K:
        raise ValueError(f"x must be [..., k] with k in [1, {MAX_K}]")
    dtype, index = _DTYPES.get(x.dtype), x.get_device()
    if dtype is None:
        raise ValueError("x must be float32, float16 or bfloat16")
    if index < 0:
        raise ValueError("quantisation runs on a HIP device")
    rows = x if len(shape) == 2 and (x.stride(1) == 1 or width == 1) else _rows(x, width)
    tokens, device = rows.shape[0], rows.device
    y = torch.empty((tokens, width), dtype=torch.int8, device=device)
    scale = torch.empty(tokens, dtype=torch.float32, device=device)
    if tokens:
        _launch(index, _pack(0, rows.data_ptr(), 0, y.data_ptr(), scale.data_ptr(), 0, 0, 0, 0, 0, tokens, 0, rows.stride(0), 0,
                             width, 0, 0, width, dtype, dtype, FIE_I8, 0, 0, 2, 0, 1.0, 0.0, 0.0))
    return y, scale
