"""Low-rank adapters of many requests beside a projection that they share.

    y[t] = base[t] + scale[i] * B[i] (A[i] x[t])        i = ids[t], the adapter of token t

``base`` is the shared projection's output (``fie_amd.linear.int8_linear``, or any other's); a token
without an adapter keeps it.  An ``AdapterBank`` holds the adapters of one projection, an
``AdapterPlan`` which tokens are whose, for all projections of a step.
"""

from __future__ import annotations

import struct

import torch

from . import _lib
from ._lib import FIE_BF16, FIE_F16, FIE_F32, FIE_I8
from .beam import _shared

_DTYPES = {torch.float32: FIE_F32, torch.float16: FIE_F16, torch.bfloat16: FIE_BF16}
_pack = struct.Struct(_lib.ADAPTER_ARGS).pack
_pack_plan = struct.Struct(_lib.ADAPTER_PLAN_ARGS).pack
_run = _run_plan = _size = None         # the library's entries, loaded with the first call
_raw_stream = torch._C._cuda_getCurrentRawStream
MAX_RANK = 256
MAX_ADAPTERS = 4096
MAX_TOKENS = 1 << 20
MAX_K = 131071
MAX_CHANNELS = 0x7FFFFF00


def _keep(index: int, *tensors: torch.Tensor) -> None:
    if not torch.cuda.is_current_stream_capturing():
        stream = torch.cuda.current_stream(index)
        for t in tensors:
            t.record_stream(stream)


class AdapterPlan:
    """Which tokens are whose: made by ``AdapterBank.plan``, for any bank of as many adapters."""

    def __init__(self, ids: torch.Tensor, adapters: int):
        if ids.dtype != torch.int32 or ids.ndim != 1 or ids.shape[0] > MAX_TOKENS:
            raise ValueError(f"ids must be int32 [tokens], {MAX_TOKENS} at most")
        self.index = ids.get_device()
        if self.index < 0:
            raise ValueError("adapters run on a HIP device")
        self.tokens, self.adapters = ids.shape[0], adapters
        ids = ids.contiguous()
        lib = _lib.load()
        n = lib.fie_adapter_plan_ints(self.tokens, adapters)
        if not n:
            raise ValueError(f"{self.tokens} tokens of {adapters} adapters are more than one call takes")
        self.data = torch.empty(n, dtype=torch.int32, device=ids.device)
        global _run_plan
        if _run_plan is None:
            _run_plan = _lib.launcher("fie_adapter_plan")
        _run_plan(self.index, _pack_plan(ids.data_ptr(), self.data.data_ptr(), self.tokens, adapters))
        self._made_on = _raw_stream(self.index)

    def on_stream(self) -> None:
        """Memory made on another stream is kept for this one (which waits for that one itself)."""
        if _raw_stream(self.index) != self._made_on:
            _keep(self.index, self.data)


class AdapterBank:
    """``adapters`` pairs A [rank, k], B [n, rank] of one projection, laid out for the kernels; each may
    have a smaller rank than the bank's, and is given by ``load``."""

    def __init__(self, adapters: int, k: int, n: int, rank: int, dtype: torch.dtype, device: torch.device | str):
        if not 1 <= adapters <= MAX_ADAPTERS or not 1 <= rank <= MAX_RANK:
            raise ValueError(f"adapters must be in [1, {MAX_ADAPTERS}], rank in [1, {MAX_RANK}]")
        if not 1 <= k <= MAX_K or not 1 <= n <= MAX_CHANNELS:
            raise ValueError(f"k must be in [1, {MAX_K}], n in [1, {MAX_CHANNELS}]")
        if dtype not in _DTYPES:
            raise ValueError("dtype must be float32, float16 or bfloat16")
        if torch.device(device).type != "cuda":
            raise ValueError("adapters run on a HIP device")
        self.adapters, self.k, self.n, self.rank, self.dtype = adapters, k, n, rank, dtype
        self.rank_pad, self.k_pad = -(-rank // 16) * 16, -(-k // 64) * 64
        self.a = torch.zeros((adapters, self.rank_pad, self.k_pad), dtype=dtype, device=device)
        # Channels that begin at every 128 bytes come in slowly where tiles share them (the second product, us,
        # with 16 bytes more a channel and without): 4001 x 4096 in bf16 rank 64 37 and 53, 128 138 and 179, 256
        # 263 and 339; in fp32 rank 32 32 and 35, 64 47 and 53, 256 193 and 239.  250 x 16384 of 64 adapters, each
        # read once or twice: bf16 36 and 49, 137 and 139, 272 and 278; fp32 35 and 35, 74 and 67, 366 and 293
        size = self.a.element_size()
        self.b_pitch = self.rank_pad + (16 // size if self.rank_pad * size % 128 == 0 else 0)
        self.b = torch.zeros((adapters, n, self.b_pitch), dtype=dtype, device=device)
        self.scale = torch.zeros(adapters, dtype=torch.float32, device=device)
        self.ranks = torch.zeros(adapters, dtype=torch.int32, device=device)
        self.device, self.index = self.a.device, self.a.get_device()
        self._made_on = _raw_stream(self.index)

    def on_stream(self) -> None:
        """Memory made on another stream is kept for this one (which waits for that one itself)."""
        if _raw_stream(self.index) != self._made_on:
            _keep(self.index, self.a, self.b, self.scale, self.ranks)

    def load(self, i: int, a: torch.Tensor, b: torch.Tensor, scale: float = 1.0) -> None:
        """Adapter i: a [rank, k], b [n, rank], rank up to the bank's (0: it does nothing).  On the current
        stream, as everything that reads the bank."""
        if not 0 <= i < self.adapters:
            raise ValueError(f"adapters are 0 .. {self.adapters - 1}")
        if a.ndim != 2 or b.ndim != 2 or a.shape[1] != self.k or b.shape != (self.n, a.shape[0]) or a.shape[0] > self.rank:
            raise ValueError(f"a must be [rank, {self.k}], b [{self.n}, rank], rank at most {self.rank}")
        r = a.shape[0]
        self.on_stream()
        self.a[i].zero_()
        self.b[i].zero_()
        self.a[i, :r, :self.k] = a
        self.b[i, :, :r] = b
        self.scale[i] = scale
        self.ranks[i] = r

    def plan(self, ids: torch.Tensor) -> AdapterPlan:
        """Each token's adapter, int32 [tokens] (outside [0, adapters): none)."""
        if ids.get_device() != self.index:
            raise ValueError("ids must be on the bank's device")
        return AdapterPlan(ids, self.adapters)


def adapter_linear(x: torch.Tensor, bank: AdapterBank, plan: AdapterPlan, *, x_scale: torch.Tensor | None = None,
                   base: torch.Tensor | None = None, out: torch.Tensor | None = None,
                   out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``base`` and each token's adapter's product: x [..., k] in the bank's type, or int8 with ``x_scale``
    (float32, one a token); base [..., n] in the output's type or float32 (None: 0).

    The output is in ``out_dtype``, the bank's type or float32; by default the bank's.  ``out`` [tokens, n] is
    written instead of a new tensor (unit element stride, any row stride); it may be ``base`` itself,
    else it is apart from it.
    A[i] x[t] is summed in fp32 and, with two-byte adapters, each of its numbers enters the second
    product as two of their type, together off by 2^-16 of it (bf16) or by 2^-22 of it and 2^-39 of the
    token's largest, whichever is more (fp16); that product's sums are fp32, and the result is rounded
    once.  Infinite and NaN activations give what the formula gives, for their token alone; adapters
    themselves are finite numbers.  Runs on the current stream; nothing waits for it."""
    shape, k, n, tokens, index = x.shape, bank.k, bank.n, plan.tokens, bank.index
    if not shape or shape[-1] != k or x.numel() != tokens * k:
        raise ValueError(f"x must be [..., {k}] of the plan's {tokens} tokens")
    if plan.adapters != bank.adapters:
        raise ValueError(f"the plan is of {plan.adapters} adapters, the bank of {bank.adapters}")
    if x.get_device() != index or plan.index != index:
        raise ValueError("every tensor must be on the bank's device")
    code = _DTYPES[bank.dtype]
    xs = 0
    if x.dtype == torch.int8:
        if x_scale is None or x_scale.dtype != torch.float32 or x_scale.numel() != tokens or not x_scale.is_contiguous() \
                or x_scale.get_device() != index:
            raise ValueError(f"int8 tokens need x_scale, contiguous float32 of {tokens} on the bank's device")
        x_code, xs = FIE_I8, x_scale.data_ptr()
    elif x.dtype == bank.dtype:
        if x_scale is not None:
            raise ValueError("x_scale belongs to int8 tokens")
        x_code = code
    else:
        raise ValueError(f"x must be {bank.dtype} or int8")
    if x.ndim != 2:
        x = x.reshape(tokens, k)
    if (k > 1 and x.stride(1) != 1) or (tokens > 1 and x.stride(0) < 0):
        x = x.contiguous()
    dtype = out_dtype if out_dtype is not None else out.dtype if out is not None else bank.dtype
    if dtype != bank.dtype and dtype != torch.float32:
        raise ValueError(f"out_dtype must be {bank.dtype} or float32")
    bp = b_stride = b_code = 0
    if base is not None:
        if base.shape != (*shape[:-1], n) or base.get_device() != index or (base.dtype != dtype and base.dtype != torch.float32):
            raise ValueError(f"base must be [..., {n}] in {dtype} or float32 on the bank's device")
        rows = base if base.ndim == 2 else base.reshape(tokens, n)
        if n > 1 and rows.stride(1) != 1:
            rows = rows.contiguous()
        bp, b_stride, b_code = rows.data_ptr(), rows.stride(0), _DTYPES[base.dtype]
    if out is None:
        y = torch.empty((tokens, n), dtype=dtype, device=x.device)
    else:
        if out.ndim != 2 or out.shape != (tokens, n) or out.dtype != dtype or (n > 1 and out.stride(1) != 1) \
                or (tokens > 1 and out.stride(0) < n) or out.get_device() != index:
            raise ValueError(f"out must be [{tokens}, {n}] in {dtype} with unit element stride")
        y = out
    if tokens:
        global _run, _size
        if _run is None:
            _run, _size = _lib.launcher("fie_adapter_linear"), _lib.load().fie_adapter_workspace_size
        yp, y_stride = y.data_ptr(), max(y.stride(0), n)
        if bp == yp and (base.dtype != dtype or (tokens > 1 and b_stride != y_stride)):
            raise ValueError("base and out in one place must be the same tensor")
        if bp == yp:
            b_stride = y_stride
        elif bp and out is not None:
            def part(p, stride, size):
                return p, p + ((tokens - 1) * stride + n) * size, stride * size if tokens > 1 else 0, n * size

            if _shared(part(bp, b_stride, base.element_size()), part(yp, y_stride, y.element_size())):
                raise ValueError("out must be base itself or apart from it")
        args = [x.data_ptr(), xs, bank.a.data_ptr(), bank.b.data_ptr(), bank.scale.data_ptr(), bank.ranks.data_ptr(),
                plan.data.data_ptr(), bp, yp, 0, 0, x.stride(0), b_stride, y_stride, tokens, k, n, bank.adapters, bank.rank_pad,
                bank.k_pad, bank.b_pitch, code, x_code, _DTYPES[dtype], b_code, 0]
        args[10] = _size(_pack(*args))
        room = torch.empty(args[10], dtype=torch.uint8, device=y.device)
        args[9] = room.data_ptr()
        plan.on_stream()
        bank.on_stream()
        _run(index, _pack(*args))
    return y.view(*shape[:-1], n) if out is None and len(shape) != 2 else y
