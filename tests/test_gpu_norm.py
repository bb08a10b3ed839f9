"""Block norms on an MI355X against the formulas in 64 bits.

An output is rounded once from fp32: half a unit of its type (2^-8 bf16, 2^-11 fp16, 2^-24
fp32 of the value).  The fp32 work before it adds a few 2^-24 of the largest term: a sum of
squares over at most 65536 in lanes and waves is off by less than 40 of them, and what enters
is rescaled by it, so 1e-5 of the row's largest value covers it.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from fie_amd.linear import quantize_rows
from fie_amd.norm import MAX_WIDTH, block_norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def norm64(v, kind, weight, bias, eps, offset):
    if kind == "none":
        return v
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)
    if weight is not None:
        v = v * (weight.double().cpu() + offset)
    return v if bias is None else v + bias.double().cpu()


def plain(residual, x, weight, bias=None, post_weight=None, post_bias=None, post_norm=None, gate=None, scale=1.0,
          eps=1e-6, kind="rms", weight_offset=0.0):
    r = residual.double().cpu()
    if x is not None:
        z = x.double().cpu()
        if post_norm if post_norm is not None else post_weight is not None:
            z = norm64(z, kind, post_weight, post_bias, eps, weight_offset)
        if gate is not None:
            z = z * gate.double().cpu()
        r = r + float(np.float32(scale)) * z
    return r, norm64(r, kind, weight, bias, eps, weight_offset)


def near(got, want, dtype, what):
    g, w = got.double().cpu(), want
    bound = HALF[dtype] * w.abs() * 1.01 + 1e-5 * w.abs().amax(-1, keepdim=True) + 1e-30
    if dtype == torch.float16:
        bound = bound + 2.0 ** -25           # subnormal
    bad = (g - w).abs() > bound
    assert not bad.any(), (what, int(bad.sum()), float(((g - w).abs() / bound).max()))


def make(seed, shape, dtype, rdtype):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    x, r = rnd(*shape), 3.0 * rnd(*shape)
    x[..., ::11] *= 8.0
    H = shape[-1]
    return dict(x=x.to(dtype), residual=r.to(rdtype), weight=(1.0 + 0.2 * rnd(H)).to(dtype), bias=rnd(H).to(dtype),
                post_weight=(1.0 + 0.2 * rnd(H)).to(dtype), post_bias=(0.1 * rnd(H)).to(dtype), rnd=rnd)


WIDTHS = [1, 2, 7, 8, 63, 64, 65, 511, 512, 513, 520, 2048, 2050, 4096, 4100, 8191, 8200, 16384, 16392, 40001, 65536]


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype, rdtype", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32),
                                           (torch.float32, torch.float32)])
def test_widths(width, dtype, rdtype):
    for kind in ("rms", "layer"):
        m = make(width, (5, width), dtype, rdtype)
        m.pop("rnd")
        eps = 1e-2 if width < 8 else 1e-6            # a layer norm of one or two values has no spread
        kw = dict(m, scale=0.7, eps=eps, kind=kind)
        got = block_norm(kw.pop("residual"), kw.pop("x"), kw.pop("weight"), **kw)
        r, y = plain(m["residual"], m["x"], m["weight"], m["bias"], m["post_weight"], m["post_bias"], scale=0.7,
                     eps=eps, kind=kind)
        near(got.residual, r, rdtype, (width, kind, "residual"))
        near(got.y, y, dtype, (width, kind, "y"))
        assert got.residual.dtype == rdtype and got.y.dtype == dtype


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("gate", ["none", "channel", "token", "row", "fp32"])
@pytest.mark.parametrize("kind", ["rms", "layer", "none"])
def test_parts(dtype, gate, kind):
    m = make(3, (3, 11, 1000), dtype, dtype)
    rnd = m["rnd"]
    g = dict(none=None, channel=rnd(1000).to(dtype), token=rnd(3, 11, 1000).to(dtype), row=rnd(3, 11, 1).to(dtype),
             fp32=rnd(1000))[gate]
    for post in (False, True):
        if kind == "none" and post:
            continue
        for offset in (0.0, 1.0):
            p = dict(gate=g, scale=-0.3, eps=1e-5, kind=kind, weight_offset=offset)
            weight = None if kind == "none" else m["weight"]
            if post:
                p.update(post_weight=m["post_weight"])
            got = block_norm(m["residual"], m["x"], weight, **p)
            r, y = plain(m["residual"], m["x"], weight, **p)
            near(got.residual, r, dtype, "residual")
            near(got.y, y, dtype, "y")
            assert got.y.shape == m["x"].shape and got.scale is None


def test_post_norm_without_a_weight_and_fp32_parameters():
    m = make(4, (9, 777), torch.bfloat16, torch.float32)
    w = m["weight"].float() * 1.0001
    got = block_norm(m["residual"], m["x"], w, post_norm=True, bias=m["bias"].float())
    r, y = plain(m["residual"], m["x"], w, m["bias"].float(), post_norm=True)
    near(got.residual, r, torch.float32, "residual")
    near(got.y, y, torch.bfloat16, "y")


@pytest.mark.parametrize("rdtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("out", [torch.float32, torch.float16, torch.bfloat16])
def test_residual_alone(rdtype, out):
    m = make(5, (4, 1234), out, rdtype)
    got = block_norm(m["residual"], None, m["weight"], out_dtype=out)
    assert got.residual is None
    near(got.y, plain(m["residual"], None, m["weight"])[1], out, "y")


@pytest.mark.parametrize("width", [1, 9, 64, 513, 4096, 5001, 16400, 65536])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_int8(width, dtype):
    m = make(6, (7, width), dtype, dtype)
    m["x"][3], m["residual"][3] = 0, 0
    got = block_norm(m["residual"], m["x"], m["weight"], quantize=True)
    r, y = plain(m["residual"], m["x"], m["weight"])
    s = y.abs().amax(-1) / 127
    np.testing.assert_allclose(got.scale.cpu().numpy(), s.numpy(), rtol=1e-5, atol=0)
    assert got.y.dtype == torch.int8 and got.scale[3] == 0 and not got.y[3].any()
    # half a step, and what fp32 is off by (1e-5 of the row's largest, 127 steps)
    assert ((got.y.double().cpu() * s[:, None] - y).abs() <= s[:, None] * (0.5 + 2 * 127e-5)).all()
    near(got.residual, r, dtype, "residual")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("width", [1, 17, 64, 1000, 4096, 16385])
def test_quantize_rows_is_the_ieee_quotient(dtype, width):
    gen = torch.Generator().manual_seed(width)
    x = (torch.randn(6, width, generator=gen) * torch.tensor([1.0, 1e-3, 300.0, 1e-7, 0.0, 50.0])[:, None]).to(dtype)
    x[5, 0] = float("nan")
    q, s = quantize_rows(x.to(DEV))
    v = x.float().numpy()
    want = np.nanmax(np.abs(v), axis=1) / np.float32(127)
    want = np.where(np.isnan(want), np.float32(0), want).astype(np.float32)
    np.testing.assert_array_equal(s.cpu().numpy(), want)
    with np.errstate(invalid="ignore", divide="ignore"):
        t = np.rint(v / want[:, None])
    np.testing.assert_array_equal(q.cpu().numpy(), np.where(np.isnan(t), 0, t).astype(np.int8))


@pytest.mark.parametrize("units", [1, 63, 64, 100, 190, 191, 254, 1000, 12345])
def test_quantize_rows_of_denormals(units):
    """Rows of a few 2^-149: the scale, itself a denormal, is off by up to half of itself."""
    x = (np.arange(-8, 9) * units // 8 * 2.0 ** -149).astype(np.float32)
    q, s = quantize_rows(torch.from_numpy(x[None]).to(DEV))
    scale = np.float32(np.abs(x).max()) / np.float32(127)
    assert s.cpu().numpy()[0] == scale
    want = np.clip(np.rint(x.astype(np.float64) / scale), -127, 127) if scale > 0 else np.zeros(17)
    np.testing.assert_array_equal(q.cpu().numpy()[0], want.astype(np.int8))


def test_strides_inplace_and_streams():
    H, T = 1003, 13
    m = make(8, (T, H), torch.bfloat16, torch.bfloat16)
    want = plain(m["residual"], m["x"], m["weight"], gate=m["post_weight"])

    def wide(t, pad, at):
        big = torch.full((t.shape[0], t.shape[1] + pad), float("nan"), dtype=t.dtype, device=DEV)
        big[:, at:at + t.shape[1]] = t
        return big, big[:, at:at + t.shape[1]]

    xb, x = wide(m["x"], 5, 3)
    rb, r = wide(m["residual"], 9, 1)
    got = block_norm(r, x, m["weight"], gate=m["post_weight"])
    near(got.residual, want[0], torch.bfloat16, "residual")
    near(got.y, want[1], torch.bfloat16, "y")
    got = block_norm(m["residual"].t().contiguous().t(), x, m["weight"], gate=m["post_weight"])
    near(got.y, want[1], torch.bfloat16, "y")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = block_norm(r, x, m["weight"], gate=m["post_weight"], inplace=True)
        assert got.residual is r
        near(r, want[0], torch.bfloat16, "residual")
    torch.cuda.current_stream().wait_stream(side)
    assert torch.isnan(rb[:, 0]).all() and torch.isnan(rb[:, H + 1:]).all()
    # a row shared by all tokens
    one = m["x"][:1].expand(T, H)
    near(block_norm(m["residual"], one, m["weight"]).y, plain(m["residual"], one, m["weight"])[1], torch.bfloat16, "y")


def test_no_tokens_and_unusual_values():
    for q in (False, True):
        got = block_norm(torch.empty(0, 64, device=DEV), torch.empty(0, 64, device=DEV), quantize=q)
        assert got.y.shape == (0, 64) and got.residual.shape == (0, 64)
    x = torch.randn(5, 300, device=DEV)
    x[1, 7], x[2, 7] = float("nan"), float("inf")
    x[3] *= 1e18                                       # squares near fp32's limit stay with their row
    got = block_norm(torch.zeros_like(x), x).y
    assert torch.isnan(got[1]).all() and torch.isfinite(got[[0, 3, 4]]).all()
    near(got[[0, 4]], plain(torch.zeros(2, 300), x[[0, 4]], None)[1], torch.float32, "neighbours")


def test_refusals():
    r = torch.randn(4, 64, device=DEV)
    w = torch.ones(64, device=DEV)
    for args, kw in [((r, r[:3]), {}), ((r.half(), r), {}), ((r, r, w[:63]), {}),
                     ((r, r, w.half()), {}), ((r, r, w), dict(kind="group")), ((r, r, w), dict(kind="none")),
                     ((r, r, w), dict(post_bias=w)), ((r, None, w), dict(gate=w)), ((r, None, w), dict(inplace=True)),
                     ((r, r, w), dict(gate=w[:5])), ((r, r, w), dict(gate=w.double())), ((r.double(), None), {}),
                     ((r.cpu(), None), {}), ((r, r.cpu()), {}), ((r, r, w), dict(bias=w.half())),
                     ((r, r, w), dict(out_dtype=torch.float16)), ((r, None), dict(out_dtype=torch.int8)),
                     ((torch.empty(1, MAX_WIDTH + 1, device=DEV), None), {}), ((torch.tensor(1.0, device=DEV), None), {}),
                     ((r.t().contiguous().t(), r, w), dict(inplace=True)), ((r[:1].expand(4, 64), r), dict(inplace=True))]:
        with pytest.raises(ValueError):
            block_norm(*args, **kw)


def test_large_offsets():
    """More than 2^31 elements: the last rows."""
    T, H = 2 ** 31 // 32768 + 40, 32768
    x = torch.zeros(T, H, dtype=torch.float16, device=DEV)
    gen = torch.Generator(device=DEV).manual_seed(1)
    x[-5:] = torch.randn(5, H, generator=gen, device=DEV).half()
    got = block_norm(x, x)
    r, y = plain(x[-5:], x[-5:], None)
    near(got.residual[-5:], r, torch.float16, "residual")
    near(got.y[-5:], y, torch.float16, "y")
    assert not got.y[:5].any()
    q, s = quantize_rows(x)
    assert not q[:-5].any() and s[-1] > 0 and q[-5:].abs().amax() == 127
