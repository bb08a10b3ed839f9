"""A matrix product in 8-bit integers with a scale for each token and each output channel.

    y[t, n] = x_scale[t] * w_scale[n] * sum_k x[t, k] * w[n, k]   (+ bias[n])

The sums are exact in 32 bits (k up to MAX_K; those of longer products could pass them); scaling
is fp32, rounded once to the output's type.  Weights keep nn.Linear's [channels, k] layout.
"""

from __future__ import annotations

import struct

import torch

from . import _lib
from ._lib import FIE_BF16, FIE_F16, FIE_F32
from .norm import MAX_K, quantized

_DTYPES = {torch.float32: FIE_F32, torch.float16: FIE_F16, torch.bfloat16: FIE_BF16}
_pack = struct.Struct(_lib.INT8_ARGS).pack
_run = None             # the library's entry, loaded with the first call
MAX_CHANNELS = 0x7FFFFF00


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(q, scale) of x [..., k]: scale = max|row| / 127 (float32 [rows]), q = round(row / scale) in
    int8, ties to even; a row of zeros gives 0 and scale 0, a row with a NaN 0 and scale NaN (its
    products are then NaN).  For a weight [channels, k] it gives the scales of its channels, for
    activations those of the tokens."""
    q, scale = quantized(x)
    return q if x.ndim == 2 else q.view(x.shape), scale


def _vector(t: torch.Tensor, name: str, size: int, index: int) -> int:
    """Its address, if it is a contiguous float32 of that size on that device."""
    if t.dtype != torch.float32 or t.numel() != size or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous float32 of {size}")
    if t.get_device() != index:
        raise ValueError("every tensor must be on the weight's device")
    return t.data_ptr()


def int8_linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, *,
                x_scale: torch.Tensor | None = None, bias: torch.Tensor | None = None,
                out_dtype: torch.dtype | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """x [..., k] times weight [n, k] int8, transposed, as nn.Linear does it.

    x is int8 with ``x_scale`` (float32, one a token), or float32, float16 or bfloat16, which is
    quantised for each token first.  ``out_dtype``: float32, float16 or bfloat16; by default x's own
    (bfloat16 for int8).  Rows of weights and of int8 tokens that begin at multiples of 16 bytes
    (pad those of a storage where k is none: ``w = room[:, :k]``) are read fastest; others go at their
    own addresses up to 96 tokens, and past them are laid out anew in every call.  (Tokens that are
    quantised here or by ``quantize_rows`` have rows of k bytes.)  ``out`` [tokens, n] is written instead of a new tensor: unit element
    stride, any row stride.  Runs on the current stream; nothing waits for it."""
    if weight.ndim != 2 or weight.dtype != torch.int8:
        raise ValueError("weight must be int8 [channels, k]")
    n, k = weight.shape
    shape = x.shape
    if not shape or shape[-1] != k or not 1 <= n <= MAX_CHANNELS or not 1 <= k <= MAX_K:
        raise ValueError(f"x [..., k] and weight [channels, k] must agree on k in [1, {MAX_K}]")
    index = weight.get_device()
    if index < 0:
        raise ValueError("int8_linear runs on a HIP device")
    if x.get_device() != index or (out is not None and out.get_device() != index):
        raise ValueError("every tensor must be on the weight's device")
    tokens = x.numel() // k
    ws = _vector(weight_scale, "weight_scale", n, index)
    xs = _vector(x_scale, "x_scale", tokens, index) if x_scale is not None else 0
    bs = _vector(bias, "bias", n, index) if bias is not None else 0
    if x.dtype == torch.int8:
        if x_scale is None:
            raise ValueError("int8 tokens need x_scale")
        dtype = out_dtype or torch.bfloat16
    elif x.dtype in _DTYPES:
        if x_scale is not None:
            raise ValueError("x_scale belongs to int8 tokens")
        dtype = out_dtype or x.dtype
    else:
        raise ValueError("x must be int8, float32, float16 or bfloat16")
    y_dtype = _DTYPES.get(dtype)
    if y_dtype is None:
        raise ValueError("out_dtype must be float32, float16 or bfloat16")
    if out is None:
        y, y_stride = torch.empty((tokens, n), dtype=dtype, device=weight.device), n
    else:
        if out.ndim != 2 or out.shape != (tokens, n) or out.dtype != dtype or (n > 1 and out.stride(1) != 1) \
                or (tokens > 1 and out.stride(0) < n):
            raise ValueError(f"out must be [{tokens}, {n}] in {dtype} with unit element stride")
        y, y_stride = out, max(out.stride(0), n)
    if tokens:
        if x.dtype != torch.int8:
            x, x_scale = quantized(x)
            xs = x_scale.data_ptr()
        elif len(shape) != 2:
            x = x.reshape(-1, k)
        x_stride, step = x.stride()
        if (k > 1 and step != 1) or (tokens > 1 and x_stride < k):
            x, x_stride = x.contiguous(), k
        w_stride, step = weight.stride()
        if (k > 1 and step != 1) or (n > 1 and w_stride < k):
            weight, w_stride = weight.contiguous(), k
        xp, wp, x_stride, w_stride = x.data_ptr(), weight.data_ptr(), max(x_stride, k), max(w_stride, k)
        args = [xp, wp, xs, ws, bs, y.data_ptr(), tokens, x_stride, w_stride, y_stride, n, k, y_dtype, 0, 0, 0]
        global _run
        if _run is None:
            _run = _lib.launcher("fie_int8_linear")
        if (xp | wp | x_stride | w_stride) & 15 or x_stride >= 1 << 23 or w_stride >= 1 << 23:
            args[-1] = _lib.load().fie_int8_workspace_size(_pack(*args))
            if args[-1]:
                room = torch.empty(args[-1], dtype=torch.int8, device=y.device)
                args[-2] = room.data_ptr()
        _run(index, _pack(*args))
    return y.view(*shape[:-1], n) if out is None and len(shape) != 2 else y
