"""Beams, pages and adapters without a GPU: exported functions, argument layouts, refusals.

No call here reaches a launch: each fails its checks first."""

from __future__ import annotations

import os
import re
import shutil
import struct
import subprocess

import pytest
import torch

from fie_amd import _lib, adapters, beam, pages
from fie_amd.adapters import AdapterBank
from fie_amd.beam import Beams, BeamSearch, beam_step, first_beams, reorder_states
from fie_amd.pages import CachePages

INCLUDE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
HEADER = os.path.join(INCLUDE, "fie_decode.h")


def test_library_exports_what_the_header_declares():
    declared = set(re.findall(r"^\s*(?:int|size_t)\s+(fie_\w+)\s*\(", open(HEADER).read(), re.M))
    assert declared == set(_lib.DECODE_EXPORTS)
    lib = _lib.load()
    for name in declared:
        assert hasattr(lib, name), name


BEAM = ("logits scores lengths done pool ends next_scores next_lengths next_done next_pool next_ends tokens parents history_tokens "
        "history_parents row_stride workspace workspace_bytes length_penalty requests beams vocab dtype early_stopping min_tokens pad "
        "history_steps eos_count").split() + [f"eos[{i}]" for i in range(16)] + ["max_tokens"]
PLAN = "ids plan tokens adapters".split()
ADAPTER = ("x x_scale a b scale ranks plan base y workspace workspace_bytes x_stride base_stride y_stride tokens k n adapters rank k_pad "
           "b_pitch dtype x_dtype y_dtype base_dtype reserved").split()
GROUP = "base page_stride outer_stride token_bytes count outer whole shift".split()
PAGES = ("state scratch scratch_bytes pages page rows wide parents lengths granted live src dst copies group_count").split()
STATE = "src dst src_stride dst_stride row_bytes rows".split()


def offsets(fmt):
    at, got = 0, []
    for count, code in re.findall(r"(\d*)([A-Za-z])", fmt.lstrip("@")):
        for _ in range(int(count) if count else 1):
            size = struct.calcsize(code)
            at = -(-at // size) * size
            got.append(at)
            at += size
    return got


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs a C compiler")
def test_argument_layouts_are_the_headers(tmp_path):
    kinds = [("fie_beam_args", BEAM, _lib.BEAM_ARGS), ("fie_adapter_plan_args", PLAN, _lib.ADAPTER_PLAN_ARGS),
             ("fie_adapter_args", ADAPTER, _lib.ADAPTER_ARGS),
             ("fie_pages_args", PAGES + [f"group[{i}].{f}" for i in range(8) for f in GROUP], _lib.PAGES_ARGS + _lib.GROUP_ARGS * 8),
             ("fie_states_args", "parents n count".split() + [f"state[{i}].{f}" for i in range(48) for f in STATE],
              _lib.STATES_ARGS + _lib.STATE_ARGS * 48)]
    body = "".join(f'printf("%zu ", offsetof({t}, {f}));' for t, fs, _ in kinds for f in fs)
    body += "".join(f'printf("%zu ", sizeof({t}));' for t, _, _ in kinds)
    src = tmp_path / "l.c"
    src.write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "fie_decode.h"\nint main(void) {{ {body} return 0; }}\n')
    subprocess.run(["gcc", f"-I{INCLUDE}", str(src), "-o", str(tmp_path / "l")], check=True)
    out = list(map(int, subprocess.run([str(tmp_path / "l")], check=True, capture_output=True, text=True).stdout.split()))
    want = [o for _, fs, fmt in kinds for o in offsets(fmt)]
    assert len(want) == sum(len(fs) for _, fs, _ in kinds)
    assert out == want + [struct.calcsize(fmt) for _, _, fmt in kinds]


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs a C compiler")
def test_limits_are_the_headers(tmp_path):
    names = "FIE_MAX_BEAMS FIE_MAX_EOS FIE_MAX_STATES FIE_MAX_PAGE_ROWS FIE_MAX_PAGES FIE_MAX_CACHE_GROUPS FIE_MAX_RANK FIE_MAX_ADAPTERS"
    src = tmp_path / "l.c"
    src.write_text('#include <stdio.h>\n#include "fie_decode.h"\nint main(void) {' + "".join(f'printf("%d ", {n});' for n in names.split())
                   + "return 0; }\n")
    subprocess.run(["gcc", f"-I{INCLUDE}", str(src), "-o", str(tmp_path / "l")], check=True)
    out = subprocess.run([str(tmp_path / "l")], check=True, capture_output=True, text=True).stdout.split()
    assert list(map(int, out)) == [beam.MAX_BEAMS, beam.MAX_EOS, beam.MAX_STATES, pages.MAX_ROWS, pages.MAX_PAGES, pages.MAX_GROUPS,
                                   adapters.MAX_RANK, adapters.MAX_ADAPTERS]


def refused(name, args, code, text):
    lib = _lib.load()
    assert getattr(lib, name)(args, None) == code
    assert text in lib.fie_sampler_last_error(), lib.fie_sampler_last_error()


def beam_args(**kw):
    a = {n: 0 for n in BEAM}
    a.update({n: 256 for n in BEAM[:13]}, row_stride=100, workspace=256, workspace_bytes=1 << 20, length_penalty=1.0, requests=2,
             beams=4, vocab=100)
    assert set(kw) <= set(a)
    return struct.pack(_lib.BEAM_ARGS, *{**a, **kw}.values())


@pytest.mark.parametrize("kw, code, text", [
    (dict(beams=0), _lib.FIE_E_ARG, b"beams"), (dict(beams=65), _lib.FIE_E_ARG, b"beams"), (dict(requests=-1), _lib.FIE_E_ARG, b"rows"),
    (dict(requests=1 << 14), _lib.FIE_E_ARG, b"rows"), (dict(vocab=0), _lib.FIE_E_ARG, b"vocab"),
    (dict(vocab=524289, row_stride=524289), _lib.FIE_E_ARG, b"vocab"), (dict(dtype=3), _lib.FIE_E_ARG, b"dtype"),
    (dict(row_stride=99), _lib.FIE_E_ARG, b"row_stride"), (dict(eos_count=17), _lib.FIE_E_ARG, b"eos_count"),
    (dict(eos_count=-1), _lib.FIE_E_ARG, b"eos_count"), (dict(length_penalty=float("nan")), _lib.FIE_E_ARG, b"length_penalty"),
    (dict(scores=0), _lib.FIE_E_ARG, b"NULL"), (dict(parents=0), _lib.FIE_E_ARG, b"NULL"), (dict(logits=258), _lib.FIE_E_ARG, b"aligned"),
    (dict(min_tokens=-1), _lib.FIE_E_ARG, b"min_tokens"), (dict(max_tokens=-1), _lib.FIE_E_ARG, b"max_tokens"),
    (dict(history_tokens=256), _lib.FIE_E_ARG, b"history"), (dict(history_steps=-1), _lib.FIE_E_ARG, b"history"),
    (dict(workspace=0), _lib.FIE_E_WORKSPACE, b"too small"), (dict(workspace_bytes=16), _lib.FIE_E_WORKSPACE, b"too small"),
    (dict(workspace=264), _lib.FIE_E_WORKSPACE, b"16-byte")])
def test_beam_refusals(kw, code, text):
    refused("fie_beam_step", beam_args(**kw), code, text)


def test_beam_nothing_to_do():
    lib = _lib.load()
    assert lib.fie_beam_step(beam_args(requests=0), None) == _lib.FIE_OK
    assert lib.fie_beam_step(None, None) == _lib.FIE_E_ARG
    assert lib.fie_beam_workspace_size(beam_args(requests=0)) == lib.fie_beam_workspace_size(None) == 0
    assert lib.fie_beam_workspace_size(beam_args()) == 8 * (16 + 8 * 4)


@pytest.mark.parametrize("state, text", [
    ((0, 256, 16, 16, 16, 4), b"NULL"), ((256, 0, 16, 16, 16, 4), b"NULL"), ((256, 512, 16, 16, 16, 3), b"rows"),
    ((256, 512, 16, 16, 0, 4), b"empty"), ((256, 512, 16, 15, 16, 4), b"overlap"), ((256, 512, 16, 1 << 39, 1 << 39, 4), b"one launch")])
def test_state_refusals(state, text):
    refused("fie_reorder_states", struct.pack(_lib.STATES_ARGS + _lib.STATE_ARGS, 256, 4, 1, *state), _lib.FIE_E_ARG, text)


def test_states_nothing_to_do():
    head = lambda *v: struct.pack(_lib.STATES_ARGS, *v)  # noqa: E731
    lib = _lib.load()
    assert lib.fie_reorder_states(head(0, 0, 1), None) == lib.fie_reorder_states(head(0, 4, 0), None) == _lib.FIE_OK
    for args in (head(256, -1, 0), head(256, 1, 49), head(256, 1, -1)):
        refused("fie_reorder_states", args, _lib.FIE_E_ARG, b"out of range")
    refused("fie_reorder_states", struct.pack(_lib.STATES_ARGS + _lib.STATE_ARGS, 0, 4, 1, 256, 512, 16, 16, 16, 4), _lib.FIE_E_ARG, b"parents")
    assert lib.fie_reorder_states(None, None) == _lib.FIE_E_ARG


def page_args(group=(), **kw):
    a = {n: 256 for n in PAGES}
    a.update(scratch_bytes=1 << 20, pages=20, page=4, rows=3, wide=6, copies=2, group_count=1 if group else 0)
    assert set(kw) <= set(a)
    flat = list(group) + [0] * (64 - len(group))
    return struct.pack(_lib.PAGES_ARGS + _lib.GROUP_ARGS * 8, *{**a, **kw}.values(), *flat)


@pytest.mark.parametrize("kw, code, text", [
    (dict(pages=0), _lib.FIE_E_ARG, b"pages"), (dict(pages=(1 << 21) + 1), _lib.FIE_E_ARG, b"pages"), (dict(page=0), _lib.FIE_E_ARG, b"page out"),
    (dict(page=65537), _lib.FIE_E_ARG, b"page out"), (dict(rows=0), _lib.FIE_E_ARG, b"rows"), (dict(rows=4097), _lib.FIE_E_ARG, b"rows"),
    (dict(wide=0), _lib.FIE_E_ARG, b"wide"), (dict(wide=21), _lib.FIE_E_ARG, b"wide"), (dict(state=0), _lib.FIE_E_ARG, b"state"),
    (dict(scratch=0), _lib.FIE_E_WORKSPACE, b"too small"), (dict(scratch_bytes=64), _lib.FIE_E_WORKSPACE, b"too small"),
    (dict(scratch=260), _lib.FIE_E_WORKSPACE, b"16-byte"), (dict(group_count=9), _lib.FIE_E_ARG, b"group_count"),
    (dict(group=(0, 16, 0, 16, 1, 1, 0, 0)), _lib.FIE_E_ARG, b"layout"), (dict(group=(256, 16, 0, 0, 1, 1, 0, 0)), _lib.FIE_E_ARG, b"layout"),
    (dict(group=(256, 16, 0, 16, 1, 0, 0, 0)), _lib.FIE_E_ARG, b"layout"),
    (dict(group=(256, 16, 0, 1 << 30, 1 << 20, 1 << 10, 0, 0)), _lib.FIE_E_ARG, b"too large")])
def test_page_refusals(kw, code, text):
    for name in ("fie_pages_step", "fie_pages_compact"):
        refused(name, page_args(**kw), code, text)


def test_page_sizes_and_copies():
    lib = _lib.load()
    refused("fie_pages_step", page_args(granted=0), _lib.FIE_E_ARG, b"granted")
    refused("fie_pages_copy", page_args(copies=-1), _lib.FIE_E_ARG, b"copies")
    refused("fie_pages_copy", page_args(src=0), _lib.FIE_E_ARG, b"src")
    assert lib.fie_pages_copy(page_args(copies=0, state=0, scratch=0, src=0), None) == _lib.FIE_OK
    assert lib.fie_pages_state_ints(2050, 3, 7) == 3 * 7 + 3 + 2050 + 3
    assert lib.fie_pages_state_ints(20, 3, 21) == lib.fie_pages_state_ints(0, 3, 1) == lib.fie_pages_scratch_bytes(0, 3) == 0
    assert lib.fie_pages_scratch_bytes(20, 3) % 16 == 0


def adapter_args(**kw):
    a = {n: 256 for n in ADAPTER}
    a.update(x_scale=0, base=0, workspace_bytes=1 << 30, x_stride=64, base_stride=32, y_stride=32, tokens=4, k=64, n=32, adapters=2, rank=16, k_pad=64, b_pitch=16, reserved=0,
             dtype=_lib.FIE_BF16, x_dtype=_lib.FIE_BF16, y_dtype=_lib.FIE_BF16, base_dtype=_lib.FIE_F32)
    assert set(kw) <= set(a)
    return struct.pack(_lib.ADAPTER_ARGS, *{**a, **kw}.values())


@pytest.mark.parametrize("kw, code, text", [
    (dict(tokens=-1), _lib.FIE_E_ARG, b"tokens"), (dict(tokens=(1 << 24) + 1), _lib.FIE_E_ARG, b"tokens"),
    (dict(tokens=1 << 24), _lib.FIE_E_ARG, b"tiles"), (dict(adapters=0), _lib.FIE_E_ARG, b"adapters"),
    (dict(adapters=4097), _lib.FIE_E_ARG, b"adapters"), (dict(dtype=3, x_dtype=3), _lib.FIE_E_ARG, b"type"),
    (dict(x_dtype=_lib.FIE_F16), _lib.FIE_E_ARG, b"x is in"), (dict(y_dtype=_lib.FIE_F16), _lib.FIE_E_ARG, b"y is in"),
    (dict(base=512, base_dtype=_lib.FIE_F16), _lib.FIE_E_ARG, b"y is in"), (dict(n=0), _lib.FIE_E_ARG, b"n or k"),
    (dict(k=0), _lib.FIE_E_ARG, b"n or k"), (dict(k=131072, k_pad=131072), _lib.FIE_E_ARG, b"n or k"), (dict(k_pad=65), _lib.FIE_E_ARG, b"k_pad"),
    (dict(k=65), _lib.FIE_E_ARG, b"k_pad"), (dict(rank=8), _lib.FIE_E_ARG, b"rank"), (dict(rank=272), _lib.FIE_E_ARG, b"rank"), (dict(b_pitch=8), _lib.FIE_E_ARG, b"b_pitch"), (dict(b_pitch=20), _lib.FIE_E_ARG, b"b_pitch"),
    (dict(x_stride=-1), _lib.FIE_E_ARG, b"stride"), (dict(y_stride=31), _lib.FIE_E_ARG, b"stride"), (dict(x=0), _lib.FIE_E_ARG, b"NULL"),
    (dict(plan=0), _lib.FIE_E_ARG, b"NULL"), (dict(x_scale=256), _lib.FIE_E_ARG, b"x_scale"), (dict(x_dtype=_lib.FIE_I8), _lib.FIE_E_ARG, b"x_scale"),
    (dict(b=264), _lib.FIE_E_ARG, b"16-byte"), (dict(base=256), _lib.FIE_E_ARG, b"place"),
    (dict(workspace=0), _lib.FIE_E_WORKSPACE, b"too small"), (dict(workspace_bytes=15), _lib.FIE_E_WORKSPACE, b"too small"),
    (dict(workspace=264), _lib.FIE_E_WORKSPACE, b"16-byte")])
def test_adapter_refusals(kw, code, text):
    refused("fie_adapter_linear", adapter_args(**kw), code, text)


def test_adapter_plan_refusals():
    lib = _lib.load()
    plan = lambda *v: struct.pack(_lib.ADAPTER_PLAN_ARGS, *v)  # noqa: E731
    for args, text in ((plan(0, 256, 4, 2), b"NULL"), (plan(256, 0, 4, 2), b"NULL"), (plan(256, 256, -1, 2), b"tokens"),
                       (plan(256, 256, 4, 0), b"adapters"), (plan(256, 256, 1 << 24, 1), b"tiles")):
        refused("fie_adapter_plan", args, _lib.FIE_E_ARG, text)
    assert lib.fie_adapter_plan(None, None) == lib.fie_adapter_linear(None, None) == _lib.FIE_E_ARG
    assert lib.fie_adapter_linear(adapter_args(tokens=0), None) == _lib.FIE_OK
    assert lib.fie_adapter_plan_ints(4, 0) == 0 and lib.fie_adapter_plan_ints(40, 2) == 4 + (2 + 3) * 4 + 40


def test_python_refusals_without_a_gpu():
    b = first_beams(2, 3, "cpu")
    ids = torch.zeros(3, dtype=torch.int32)
    for call in (lambda: beam_step(torch.zeros(6, 10), b), lambda: beam_step(torch.zeros(6, 10), b._replace(scores=b.scores[0])),
                 lambda: beam_step(torch.zeros(65, 10), first_beams(1, 65, "cpu")), lambda: beam_step(torch.zeros(0, 10), first_beams(1, 0, "cpu")),
                 lambda: reorder_states([torch.zeros(3, 2)], ids), lambda: reorder_states([], ids.long()), lambda: BeamSearch("cpu", 1, 2, max_tokens=4),
                 lambda: BeamSearch("cuda:0", 0, 2, max_tokens=4), lambda: BeamSearch("cuda:0", 1, 65, max_tokens=4),
                 lambda: BeamSearch("cuda:0", 1, 2, max_tokens=0), lambda: CachePages(4, 2, 1, 2, "cpu"), lambda: CachePages(0, 2, 1, 2, "cuda:0"),
                 lambda: CachePages(4, 0, 1, 2, "cuda:0"), lambda: CachePages(4, 2, 0, 2, "cuda:0"), lambda: CachePages(4, 2, 1, 5, "cuda:0"),
                 lambda: CachePages(4, 2, 4097, 2, "cuda:0"), lambda: AdapterBank(1, 4, 4, 4, torch.float32, "cpu"),
                 lambda: AdapterBank(0, 4, 4, 4, torch.float32, "cuda:0"), lambda: AdapterBank(1, 0, 4, 4, torch.float32, "cuda:0"),
                 lambda: AdapterBank(1, 4, 4, 0, torch.float32, "cuda:0"), lambda: AdapterBank(1, 4, 4, 4, torch.int8, "cuda:0")):
        with pytest.raises(ValueError):
            call()


def test_first_beams():
    b = first_beams(3, 2, "cpu")
    assert isinstance(b, Beams) and b.scores.tolist() == [[0.0, float("-inf")]] * 3 and not b.done.any() and not b.lengths.any()
    assert (b.pool == float("-inf")).all() and (b.ends == -1).all()
