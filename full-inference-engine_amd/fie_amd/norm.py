"""Block norms: the end of one block and the norm in front of the next, in one pass.

    z = gate * post_norm(x)
    r = residual + scale * z
    y = norm(r)

with the norm over the last dimension (RMS or layer), everything in fp32 between the loads and
the stores; ``y`` optionally in 8-bit integers with a scale for each token, as
``fie_amd.linear.int8_linear`` takes it.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _lib
from ._lib import FIE_BF16, FIE_F16, FIE_F32, FIE_I8, NormArgs

_DTYPES = {torch.float32: FIE_F32, torch.float16: FIE_F16, torch.bfloat16: FIE_BF16}
_KINDS = {"rms": 0, "layer": 1, "none": 2}
MAX_WIDTH = 65536


class BlockNorm(NamedTuple):
    residual: torch.Tensor | None       # residual + scale * z, in the residual's type
    y: torch.Tensor                     # its norm: x's type, or int8
    scale: torch.Tensor | None          # float32 [tokens] with int8


def _rows(t: torch.Tensor, width: int) -> torch.Tensor:
    """[tokens, width] with unit element stride (a copy where the view has none)."""
    if t.ndim != 2:
        t = t.reshape(-1, width)
    return t if t.stride(1) == 1 or width == 1 else t.contiguous()


def _vector(t: torch.Tensor | None, name: str, width: int, dtype: torch.dtype, f32: list) -> int | None:
    if t is None:
        return None
    if t.ndim != 1 or t.shape[0] != width or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous vector of {width}")
    if t.dtype != dtype and t.dtype != torch.float32:
        raise ValueError(f"{name} must be in {dtype} or float32")
    f32.append(t.dtype == torch.float32)
    return t.data_ptr()


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
    shape, width = residual.shape, residual.shape[-1] if residual.ndim else 0
    if residual.ndim < 1 or not 1 <= width <= MAX_WIDTH:
        raise ValueError(f"residual must be [..., width] with width in [1, {MAX_WIDTH}]")
    if residual.dtype not in _DTYPES:
        raise ValueError("residual must be float32, float16 or bfloat16")
    if kind not in _KINDS:
        raise ValueError("kind must be 'rms', 'layer' or 'none'")
    dtype = residual.dtype if x is None else x.dtype
    if x is None:
        dtype = out_dtype if out_dtype is not None else dtype
        if gate is not None or post_norm or post_weight is not None or post_bias is not None or inplace:
            raise ValueError("gate, post norm and inplace need x")
    elif x.shape != shape:
        raise ValueError("x and residual must have one shape")
    elif x.dtype not in _DTYPES or residual.dtype not in (x.dtype, torch.float32):
        raise ValueError("x must be float32, float16 or bfloat16, and residual in its type or float32")
    elif out_dtype is not None and out_dtype != dtype:
        raise ValueError("out_dtype is x's type")
    if dtype not in _DTYPES:
        raise ValueError("out_dtype must be float32, float16 or bfloat16")
    post = post_norm if post_norm is not None else post_weight is not None
    if kind == "none" and (post or weight is not None or bias is not None):
        raise ValueError("kind 'none' takes no norm parameters")
    if not post and (post_weight is not None or post_bias is not None):
        raise ValueError("post parameters without post_norm")
    device = residual.device
    if device.type != "cuda":
        raise ValueError("block_norm runs on a HIP device")
    for t in (x, weight, bias, post_weight, post_bias, gate):
        if t is not None and t.device != device:
            raise ValueError("every tensor must be on the residual's device")

    a = NormArgs()
    f32: list = []
    a.weight = _vector(weight, "weight", width, dtype, f32)
    a.bias = _vector(bias, "bias", width, dtype, f32)
    a.post_weight = _vector(post_weight, "post_weight", width, dtype, f32)
    a.post_bias = _vector(post_bias, "post_bias", width, dtype, f32)
    if f32 and any(f32) != all(f32):
        raise ValueError("weights and biases must share one type")
    a.weight_f32 = bool(f32) and f32[0]
    res = _rows(residual, width)
    tokens = res.shape[0]
    a.residual, a.residual_stride, a.residual_dtype = res.data_ptr(), res.stride(0), _DTYPES[res.dtype]
    a.tokens, a.width, a.x_dtype = tokens, width, _DTYPES[dtype]
    new = None
    if x is not None:
        xs = _rows(x, width)
        a.x, a.x_stride = xs.data_ptr(), xs.stride(0)
        if inplace:
            if res.data_ptr() != residual.data_ptr() or (tokens > 1 and res.stride(0) < width):
                raise ValueError("inplace needs a residual with unit element stride and rows that do not overlap")
            new = res
        else:
            new = torch.empty((tokens, width), dtype=res.dtype, device=device)
        a.residual_out, a.residual_out_stride = new.data_ptr(), new.stride(0)
        if gate is not None:
            if gate.dtype != dtype and gate.dtype != torch.float32:
                raise ValueError(f"gate must be in {dtype} or float32")
            if gate.shape == (width,):
                g = gate.contiguous()
                a.gate_stride, a.gate_step = 0, 1
            elif gate.shape == shape:
                g = _rows(gate, width)
                a.gate_stride, a.gate_step = g.stride(0), 1
            elif gate.shape == (*shape[:-1], 1):
                g = gate.reshape(-1)
                a.gate_stride, a.gate_step = g.stride(0), 0
            else:
                raise ValueError("gate must be [width], x's shape, or x's shape with a last dimension of 1")
            a.gate, a.gate_f32 = g.data_ptr(), gate.dtype == torch.float32
    y = torch.empty((tokens, width), dtype=torch.int8 if quantize else dtype, device=device)
    a.y, a.y_stride, a.y_dtype = y.data_ptr(), width, FIE_I8 if quantize else a.x_dtype
    y_scale = None
    if quantize:
        y_scale = torch.empty(tokens, dtype=torch.float32, device=device)
        a.y_scale = y_scale.data_ptr()
    a.kind, a.post_norm = _KINDS[kind], post
    a.scale, a.eps, a.weight_offset = scale, eps, weight_offset
    if tokens:
        lib = _lib.load()
        with _lib.on_device(device):
            _lib.check(lib.fie_block_norm(ctypes.byref(a), torch.cuda.current_stream(device).cuda_stream), "fie_block_norm")
    return BlockNorm(residual if inplace else new if new is None else new.view(shape), y.view(shape), y_scale)
