"""The operators' host side on the CPU: exported functions, argument layouts, refusals.

No call here reaches a launch: each fails its checks first."""

from __future__ import annotations

import ctypes
import os
import re
import shutil
import struct
import subprocess
from collections import OrderedDict

import numpy as np
import pytest
import torch

from fie_amd import _lib
from fie_amd.batching.sampler import SEEDED_STREAM, SHARED_STREAM, BatchedSampler
from fie_amd.linear import MAX_K, int8_linear, quantize_rows
from fie_amd.norm import MAX_WIDTH, block_norm
from fie_amd.runtime.sampling import SamplingParams
from fie_amd.verify import MAX_DRAFTS, DraftVerifier

INCLUDE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")


def test_library_exports_the_operators():
    text = open(os.path.join(INCLUDE, "fie_ops.h")).read()
    declared = set(re.findall(r"^\s*(?:int|size_t)\s+(fie_\w+)\s*\(", text, re.M))
    assert declared == set(_lib.OPS_EXPORTS)
    lib = _lib.load()
    for name in declared:
        assert hasattr(lib, name), name


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs a C compiler")
def test_argument_layouts_are_the_headers(tmp_path):
    """Every field of the structures where the binding puts it."""
    names = dict(
        fie_norm_args="x residual residual_out y y_scale weight bias post_weight post_bias gate tokens x_stride "
                      "residual_stride residual_out_stride y_stride gate_stride gate_step width x_dtype residual_dtype "
                      "y_dtype weight_f32 gate_f32 kind post_norm scale eps weight_offset",
        fie_int8_args="x w x_scale w_scale bias y m x_stride w_stride y_stride n k y_dtype reserved workspace workspace_bytes",
        fie_verify_args=" ".join(n for n, _ in _lib.VerifyArgs._fields_))
    body = "".join(f'printf("%zu ", offsetof({t}, {f}));' for t, fs in names.items() for f in fs.split())
    body += "".join(f'printf("%zu ", sizeof({t}));' for t in names)
    src = tmp_path / "l.c"
    src.write_text(f'#include <stdio.h>\n#include "fie_ops.h"\nint main(void) {{ {body} return 0; }}\n')
    subprocess.run(["gcc", f"-I{INCLUDE}", str(src), "-o", str(tmp_path / "l")], check=True)
    out = list(map(int, subprocess.run([str(tmp_path / "l")], check=True, capture_output=True, text=True).stdout.split()))

    def offsets(fmt):
        at, got = 0, []
        for count, code in re.findall(r"(\d*)([A-Za-z])", fmt.lstrip("@")):
            for _ in range(int(count) if count else 1):
                size = struct.calcsize(code)
                at = -(-at // size) * size
                got.append(at)
                at += size
        return got

    want = offsets(_lib.NORM_ARGS) + offsets(_lib.INT8_ARGS)
    want += [getattr(_lib.VerifyArgs, n).offset for n, _ in _lib.VerifyArgs._fields_]
    want += [struct.calcsize(_lib.NORM_ARGS), struct.calcsize(_lib.INT8_ARGS), ctypes.sizeof(_lib.VerifyArgs)]
    assert out == want


def int8_args(**kw):
    a = dict(x=256, w=512, x_scale=16, w_scale=16, bias=0, y=256, m=4, x_stride=64, w_stride=64, y_stride=32, n=32, k=64,
             y_dtype=_lib.FIE_BF16, reserved=0, workspace=0, workspace_bytes=0)
    assert set(kw) <= set(a)
    return struct.pack(_lib.INT8_ARGS, *{**a, **kw}.values())


@pytest.mark.parametrize("kw, code, text", [
    (dict(m=-1), _lib.FIE_E_ARG, b"sizes"), (dict(n=0), _lib.FIE_E_ARG, b"sizes"),
    (dict(n=2 ** 31 - 1, y_stride=2 ** 31), _lib.FIE_E_ARG, b"sizes"), (dict(k=0), _lib.FIE_E_ARG, b"k out"),
    (dict(k=MAX_K + 1), _lib.FIE_E_ARG, b"k out"), (dict(y_dtype=3), _lib.FIE_E_ARG, b"dtype"),
    (dict(x_stride=63), _lib.FIE_E_ARG, b"stride"), (dict(w_stride=1), _lib.FIE_E_ARG, b"stride"),
    (dict(y_stride=31), _lib.FIE_E_ARG, b"stride"), (dict(x=0), _lib.FIE_E_ARG, b"NULL"), (dict(y=0), _lib.FIE_E_ARG, b"NULL"),
    (dict(x_scale=0), _lib.FIE_E_ARG, b"NULL"), (dict(m=1 << 30, n=1 << 30, y_stride=1 << 30), _lib.FIE_E_ARG, b"too large"),
    (dict(m=200, x=257), _lib.FIE_E_WORKSPACE, b"unaligned"),
    (dict(m=200, w_stride=65, workspace=256, workspace_bytes=100), _lib.FIE_E_WORKSPACE, b"unaligned"),
    (dict(m=200, w_stride=65, workspace=257, workspace_bytes=1 << 20), _lib.FIE_E_WORKSPACE, b"16-byte"),
])
def test_int8_refusals(kw, code, text):
    lib = _lib.load()
    assert lib.fie_int8_linear(int8_args(**kw), None) == code
    assert text in lib.fie_sampler_last_error()
    assert lib.fie_int8_linear(None, None) == _lib.FIE_E_ARG


def test_int8_workspace_size():
    lib = _lib.load()
    size = lambda **kw: lib.fie_int8_workspace_size(int8_args(**kw))  # noqa: E731
    assert size() == size(m=100000) == size(m=0, x=1) == 0
    assert size(m=200, x=1) == 200 * 128                     # rows of whole 128-byte stages
    assert size(m=200, w_stride=67) == 32 * 128
    assert size(m=200, x_stride=200, w=1, k=129, w_stride=160) == (200 + 32) * 256
    assert size(m=16, x=1, w=1) == 0                          # few tokens go as they are
    assert lib.fie_int8_linear(int8_args(m=0), None) == _lib.FIE_OK


def norm_args(**kw):
    a = dict(x=256, residual=256, residual_out=256, y=256, y_scale=0, weight=0, bias=0, post_weight=0, post_bias=0, gate=0,
             tokens=4, x_stride=64, residual_stride=64, residual_out_stride=64, y_stride=64, gate_stride=0, gate_step=0,
             width=64, x_dtype=_lib.FIE_BF16, residual_dtype=_lib.FIE_BF16, y_dtype=_lib.FIE_BF16, weight_f32=0, gate_f32=0,
             kind=0, post_norm=0, scale=1.0, eps=1e-6, weight_offset=0.0)
    assert set(kw) <= set(a)
    return struct.pack(_lib.NORM_ARGS, *{**a, **kw}.values())


@pytest.mark.parametrize("kw, text", [
    (dict(tokens=-1), b"tokens"), (dict(width=0), b"width"), (dict(width=MAX_WIDTH + 1), b"width"), (dict(x_dtype=3), b"dtype"),
    (dict(residual_dtype=7), b"dtype"), (dict(residual_dtype=_lib.FIE_F16), b"residual is in"),
    (dict(y_dtype=_lib.FIE_F32), b"y is in"), (dict(kind=3), b"kind"), (dict(post_norm=1, x=0), b"post_norm"),
    (dict(post_norm=1, kind=2), b"post_norm"), (dict(gate=16, x=0), b"gate"), (dict(gate=16, gate_step=2), b"gate"),
    (dict(residual=0), b"residual is NULL"), (dict(y_dtype=_lib.FIE_I8), b"y_scale"), (dict(y=0, residual_out=0), b"no output"),
])
def test_norm_refusals(kw, text):
    lib = _lib.load()
    assert lib.fie_block_norm(norm_args(**kw), None) == _lib.FIE_E_ARG
    assert text in lib.fie_sampler_last_error()
    assert lib.fie_block_norm(None, None) == _lib.FIE_E_ARG
    assert lib.fie_block_norm(norm_args(tokens=0), None) == _lib.FIE_OK


def test_verify_refusals():
    lib = _lib.load()

    def call(rows=5, vocab=100, sampler=None, **kw):
        a = _lib.SamplerArgs()
        a.dtype, a.rows, a.vocab, a.row_stride = _lib.FIE_F32, rows, vocab, vocab
        for f in ("logits", "tokens", "scale", "top_k", "top_p", "min_p", "flags", "uniform"):
            setattr(a, f, 256)
        v = _lib.VerifyArgs()
        v.requests, v.max_drafts, v.draft_stride = 2, 2, vocab
        for f in ("draft_offsets", "draft_ids", "draft_probs", "tokens", "accepted"):
            setattr(v, f, 256)
        for k, x in (sampler or {}).items():
            setattr(a, k, x)
        for k, x in kw.items():
            setattr(v, k, x)
        ws = _lib.Workspace(256, 16, rows, vocab)                # too small: nothing gets past it
        return lib.fie_sampler_verify(ctypes.byref(a), ctypes.byref(v), ctypes.byref(ws), None), lib.fie_sampler_last_error()

    for kw, text in ((dict(requests=-1), b"requests"), (dict(max_drafts=-1), b"max_drafts"), (dict(max_drafts=MAX_DRAFTS + 1), b"max_drafts"),
                     (dict(requests=6), b"rows"), (dict(max_drafts=1), b"rows"), (dict(draft_ids=None), b"draft_ids"),
                     (dict(draft_dtype=5), b"dtype"), (dict(draft_stride=99), b"draft_stride"), (dict(draws=1), b"vocabulary"),
                     (dict(tokens=None), b"NULL"), (dict(accepted=None), b"NULL"), (dict(draft_offsets=None), b"NULL"),
                     (dict(sampler=dict(logits=None)), b"NULL"), (dict(sampler=dict(row_stride=9)), b"row_stride")):
        code, message = call(**kw)
        assert code == _lib.FIE_E_ARG and text in message, (kw, message)
    code, message = call()
    assert code == _lib.FIE_E_WORKSPACE and b"too small" in message
    assert lib.fie_sampler_verify(None, None, None, None) == _lib.FIE_E_ARG


def test_python_refusals_without_a_gpu():
    x = torch.zeros(2, 8)
    for call in (lambda: block_norm(x), lambda: quantize_rows(x),
                 lambda: int8_linear(x.to(torch.int8), torch.zeros(3, 8, dtype=torch.int8), torch.ones(3), x_scale=torch.ones(2))):
        with pytest.raises(ValueError, match="HIP device"):
            call()
    v, one = DraftVerifier("cuda:0"), [SamplingParams(temperature=1.0)]
    for args in ((one, [1, 2], 10), (one, [-1], 10), (one, [MAX_DRAFTS + 1], 10), (one, [1], 0),
                 ([SamplingParams(logprobs=0)], [1], 10), ([SamplingParams(presence_penalty=1.0)], [1], 10, [[1]])):
        with pytest.raises(ValueError):
            v.plan(*args)


def test_verification_draws_follow_the_streams_of_sample():
    """Row keys of a verification: a seeded request's next draws, the shared stream's in row
    order, nothing for greedy requests."""
    s = BatchedSampler.__new__(BatchedSampler)          # the host's part alone
    s._shared_key, s._shared_draws, s._seeded, s._max_generators = 11, 0, OrderedDict(), 8
    params = [SamplingParams(temperature=1.0), SamplingParams(), SamplingParams(temperature=1.0, seed=4),
              SamplingParams(temperature=0.5)]
    keys = s._verify_keys(params, [1, 2, 2, 0], ["a", "b", "c", "d"])
    shared = lambda n: [11, SHARED_STREAM, n]  # noqa: E731
    own = lambda n: [4, SEEDED_STREAM, n]  # noqa: E731
    want = [shared(1), shared(2), [0] * 3, [0] * 3, [0] * 3, own(1), own(2), own(3), shared(3)]
    np.testing.assert_array_equal(keys, np.array(want, np.uint64))
    # sample() goes on from there
    np.testing.assert_array_equal(s._draw_keys(params, ["a", "b", "c", "d"]),
                                  np.array([shared(4), [0] * 3, own(4), shared(5)], np.uint64))
