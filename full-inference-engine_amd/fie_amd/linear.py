"""A matrix product in 8-bit integers with a scale for each token and each output channel.

    y[t, n] = x_scale[t] * w_scale[n] * sum_k x[t, k] * w[n, k]   (+ bias[n])

The sums are exact in 32 bits; scaling is fp32, rounded once to the output's type.  Weights keep
nn.Linear's [channels, k] layout.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import FIE_BF16, FIE_F16, FIE_F32, Int8Args
from .norm import block_norm

_DTYPES = {torch.float32: FIE_F32, torch.float16: FIE_F16, torch.bfloat16: FIE_BF16}
MAX_K = 131071          # the sums of longer products could pass 32 bits


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(q, scale) of x [..., k]: scale = max|row| / 127 (float32 [rows]), q = round(row / scale) in
    int8, ties to even; a row of zeros gives 0 and scale 0.  For a weight [channels, k] it gives
    the scales of its channels, for activations those of the tokens."""
    got = block_norm(x, kind="none", quantize=True)
    return got.y, got.scale


def int8_linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, *,
                x_scale: torch.Tensor | None = None, bias: torch.Tensor | None = None,
                out_dtype: torch.dtype | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """x [..., k] times weight [n, k] int8, transposed, as nn.Linear does it.

    x is int8 with ``x_scale`` (float32, one a token), or float32, float16 or bfloat16, which is
    quantised for each token first.  ``out_dtype``: float32, float16 or bfloat16; by default x's own
    (bfloat16 for int8).  Weights whose rows begin at multiples of 16 bytes are read in place at
    any number of tokens (pad the rows of a storage: ``w = room[:, :k]``); others are laid out anew
    in every call past 32 tokens.  ``out`` [tokens, n] is written instead of a new tensor: unit element
    stride, any row stride.  Runs on the current stream; nothing waits for it."""
    if weight.ndim != 2 or weight.dtype != torch.int8:
        raise ValueError("weight must be int8 [channels, k]")
    n, k = weight.shape
    if x.ndim < 1 or x.shape[-1] != k or n < 1 or not 1 <= k <= MAX_K:
        raise ValueError(f"x [..., k] and weight [channels, k] must agree on k in [1, {MAX_K}]")
    device = weight.device
    if device.type != "cuda":
        raise ValueError("int8_linear runs on a HIP device")
    for t in (x, weight_scale, x_scale, bias, out):
        if t is not None and t.device != device:
            raise ValueError("every tensor must be on the weight's device")
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
    if dtype not in _DTYPES:
        raise ValueError("out_dtype must be float32, float16 or bfloat16")
    shape = x.shape[:-1]
    tokens = x.numel() // k
    for t, name, size in ((weight_scale, "weight_scale", n), (bias, "bias", n), (x_scale, "x_scale", tokens)):
        if t is not None and (t.dtype != torch.float32 or t.numel() != size or not t.is_contiguous()):
            raise ValueError(f"{name} must be contiguous float32 of {size}")
    if out is None:
        y = torch.empty((tokens, n), dtype=dtype, device=device)
    else:
        if out.ndim != 2 or out.shape != (tokens, n) or out.dtype != dtype or (n > 1 and out.stride(1) != 1) \
                or (tokens > 1 and out.stride(0) < n):
            raise ValueError(f"out must be [{tokens}, {n}] in {dtype} with unit element stride")
        y = out
    if tokens:
        if x.dtype != torch.int8:
            x, x_scale = quantize_rows(x)
        x = x if x.ndim == 2 else x.reshape(-1, k)
        if (k > 1 and x.stride(1) != 1) or (tokens > 1 and x.stride(0) < k):
            x = x.contiguous()
        if (k > 1 and weight.stride(1) != 1) or (n > 1 and weight.stride(0) < k):
            weight = weight.contiguous()
        a = Int8Args()
        a.x, a.w, a.x_scale, a.w_scale = x.data_ptr(), weight.data_ptr(), x_scale.data_ptr(), weight_scale.data_ptr()
        a.bias = None if bias is None else bias.data_ptr()
        a.y, a.y_dtype = y.data_ptr(), _DTYPES[dtype]
        a.m, a.n, a.k = tokens, n, k
        a.x_stride, a.w_stride, a.y_stride = max(x.stride(0), k), max(weight.stride(0), k), max(y.stride(0), n)
        lib = _lib.load()
        if (a.x | a.w | a.x_stride | a.w_stride) & 15 or max(a.x_stride, a.w_stride) >= 1 << 23:
            a.workspace_bytes = lib.fie_int8_workspace_size(ctypes.byref(a))
            room = torch.empty(a.workspace_bytes, dtype=torch.int8, device=device)
            a.workspace = room.data_ptr() if a.workspace_bytes else None
        with _lib.on_device(device):
            _lib.check(lib.fie_int8_linear(ctypes.byref(a), torch.cuda.current_stream(device).cuda_stream),
                       "fie_int8_linear")
    return y.view(*shape, n) if out is None else out
