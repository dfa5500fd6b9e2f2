"""The dense feed-forward on 8-bit weights and activations against its definition in 64 bits.

Inputs are whole numbers of up to three bits whose blocks' scales are powers of two: 8 bits hold
them, and the gate and up sums are exact.  The hidden activations then differ from the
definition's only where their quotient by the scale is within the f32 error of SwiGLU of the
middle of two e4m3: there a step of e4m3 is allowed.
"""
import numpy as np
import pytest
import torch

import nomas_moe as nm
import _fp8 as F

pytestmark = pytest.mark.gpu

PATH = "blocks.0.mlp"


def whole(g, rows, cols, unit):
    """Whole numbers in [-7, 7] times unit; every 128 columns of a row hold a 7."""
    t = torch.randint(-7, 8, (rows, cols), generator=g, dtype=torch.float64)
    t[:, ::128] = 7
    return t * unit


def case(rows, D, H, seed):
    g = torch.Generator().manual_seed(seed)
    x = whole(g, rows, D, 2.0 ** -2)
    w = {"gate": whole(g, H, D, 2.0 ** -7), "up": whole(g, H, D, 2.0 ** -6), "down": whole(g, D, H, 2.0 ** -6)}
    b = {n: torch.randint(-8, 9, (v.shape[0],), generator=g, dtype=torch.float64) / 16 for n, v in w.items()}
    return x, w, b


def layer_of(w, b, dtype):
    t = {}
    for n in w:
        t[f"{PATH}.{n}.weight"] = w[n].float().numpy()
        t[f"{PATH}.{n}.bias"] = b[n].float().numpy()
    H, D = w["gate"].shape
    layer = nm.FeedForward.from_source(nm.Weights.tensors_(t, dtype), PATH, D, H)
    layer.quantize()
    return layer


def wanted(x, w, b, dtype):
    """(y, bound) in f64."""
    H = w["gate"].shape[0]
    for t in (x, w["gate"], w["up"], w["down"]):
        q, s = F.quantize(t, t is not x)
        assert torch.equal(q * F.expand(s, *t.shape, t is not x), t)  # 8 bits hold it
    g, u = x @ w["gate"].T + b["gate"], x @ w["up"].T + b["up"]
    h = g / (1 + torch.exp(-g)) * u
    # exp's argument and its own error, the sum, the reciprocal, two products, the scale and its quotient
    eh = (g.abs() + 16) * F.F32 * h.abs() + 2.0 ** -140
    q, s = F.quantize(h, False)
    each = F.expand(s, *h.shape, False)
    v, e = (h / each).abs(), eh / each + 2 * F.F32 * (h / each).abs()
    lo, hi = F.nearest((v - e).clamp(min=0)), F.nearest((v + e).clamp(max=448))
    hq = q * each
    # (the scale itself may be off by the error of the block's largest value)
    ehq = (hi - lo) * each + 24 * F.F32 * hq.abs()
    y, mag = hq @ w["down"].T + b["down"], (hq.abs() + ehq) @ w["down"].abs().T + b["down"].abs()
    e = ehq @ w["down"].abs().T
    return y, e + F.product_bound(y.abs() + e, mag, H, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,D,H", [
    (1, 8, 1), (1, 64, 100), (3, 136, 257), (16, 256, 512), (17, 1000, 130), (40, 256, 384), (64, 512, 128), (128, 264, 640),
    (129, 256, 128), (300, 392, 1000), (1000, 512, 2048), (3100, 256, 2304),
])
def test_forward(rows, D, H, dtype):
    x, w, b = case(rows, D, H, rows + D + H)
    layer = layer_of(w, b, dtype)
    big = torch.full((rows * D + 64,), 7.0, dtype=dtype, device="cuda")
    y = layer.forward_fp8(x.to(dtype).cuda(), out=big[:rows * D].view(rows, D))
    assert bool((big[rows * D:] == 7.0).all())
    want, off = wanted(x, w, b, dtype)
    assert bool(((y.cpu().double() - want).abs() <= off).all())


@pytest.mark.parametrize("rows", [5, 200])
def test_against_the_operators_it_is_made_of(rows):
    """quantize_fp8 and matmul_fp8 by hand, on random values; a 16-bit rounding of gate and up between."""
    g = torch.Generator().manual_seed(rows)
    D, H = 384, 640
    w = {n: torch.randn(*s, generator=g, dtype=torch.float64) * s[1] ** -0.5
         for n, s in (("gate", (H, D)), ("up", (H, D)), ("down", (D, H)))}
    w = {n: v.bfloat16().double() for n, v in w.items()}
    b = {n: (torch.randn(v.shape[0], generator=g) * 0.1).bfloat16().double() for n, v in w.items()}
    layer = layer_of(w, b, torch.bfloat16)
    x = torch.randn(rows, D, generator=g).bfloat16().cuda()
    y = layer.forward_fp8(x)
    q = {n: nm.quantize_fp8(v.bfloat16().cuda(), square=True) for n, v in w.items()}
    a = nm.quantize_fp8(x)
    gate, up = (nm.matmul_fp8(*a, *q[n], b[n].cuda(), dtype=torch.float32) for n in ("gate", "up"))
    h = nm.quantize_fp8(gate / (1 + torch.exp(-gate)) * up)
    z = nm.matmul_fp8(*h, *q["down"], b["down"].cuda(), dtype=torch.float32)
    # the gate and up sums differ by 1.4e-5 of their size (fp8_gemm's instructions): of the hidden values, at a
    # spacing of 2^-4 to 2^-3, a share of 2.2e-4 to 4.5e-4 lands a step away: up to 2.6e-3 of the 2-norm, and
    # half a step of bf16, 2^-8 at most
    assert float((y.float() - z).norm() / z.norm()) <= 2.6e-3 + 2.0 ** -8


def test_calls_in_a_row_streams_and_capture():
    x, w, b = case(260, 256, 384, 1)
    layer = layer_of(w, b, torch.bfloat16)
    xd = x.bfloat16().cuda()
    plain = layer.forward(xd)
    want = layer.forward_fp8(xd)
    assert torch.equal(layer.forward_fp8(xd[:10]), layer.forward_fp8(xd[:10]))
    assert torch.equal(layer.forward_fp8(xd.view(2, 130, 256)), want.view(2, 130, 256))
    y = xd.clone()
    assert torch.equal(layer.forward_fp8(y, out=y), want)
    assert torch.equal(layer.forward(xd), plain)
    assert layer.forward_fp8(xd[:0]).shape == (0, 256)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    outs = []
    for _ in range(5):
        outs.append(layer.forward_fp8(xd))
        with torch.cuda.stream(s):
            outs.append(layer.forward_fp8(xd))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    for n in (10, 260):
        xc = xd[:n].clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            y = layer.forward_fp8(xc)
        for seed in range(3):
            xc.copy_(torch.randn(n, 256, generator=torch.Generator().manual_seed(seed)))
            eager = layer.forward_fp8(xc)
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, eager)


def test_states_refused():
    x, w, b = case(3, 64, 96, 1)
    t = {f"{PATH}.{n}.{k}": v[n].float().numpy() for n in w for k, v in (("weight", w), ("bias", b))}
    layer = nm.FeedForward.from_source(nm.Weights.tensors_(t, "bf16"), PATH, 64, 96)
    xd = x.bfloat16().cuda()
    with pytest.raises(nm.NomasError, match="quantize it first"):
        layer.forward_fp8(xd)
    layer.quantize()
    with pytest.raises(nm.NomasError, match="dtype"):
        layer.forward_fp8(xd.float())
    with pytest.raises(nm.NomasError, match="last dim"):
        layer.forward_fp8(xd[:, :32])
    with pytest.raises(nm.NomasError, match="GPU"):
        layer.forward_fp8(xd.cpu())
    f32 = nm.FeedForward.from_source(nm.Weights.tensors_(t, "f32"), PATH, 64, 96)
    with pytest.raises(nm.InvalidConfig, match="f32"):
        f32.quantize()


def test_a_graph_outlives_its_workspace():
    """A call of more rows takes a new workspace; a graph captured before keeps the old one."""
    x, w, b = case(700, 256, 384, 2)
    layer = layer_of(w, b, torch.bfloat16)
    xd = x.bfloat16().cuda()
    small = xd[:40].clone()
    want = layer.forward_fp8(small)
    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        y = layer.forward_fp8(small)
    for rows in (300, 700):
        whole = layer.forward_fp8(xd[:rows])
        torch.cuda.synchronize()
        y.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
        assert torch.equal(layer.forward_fp8(xd[:rows]), whole)


@pytest.mark.parametrize("rows,D,H", [(515, 96, 2093), (41, 136, 640), (932, 912, 1805)])
def test_f16_keeps_its_accuracy(rows, D, H):
    """On values of every kind the error is the outputs' rounding, at most 2^-11 of each, and that of
    the hidden values whose rounding to 8 bits falls the other way.  An error of r of a value makes
    2 r / 2^-4 of the roundings do so, each by 2^-4 of the value: with r = 40 * 2^-24, well over what an f32
    sum of a thousand terms, SwiGLU and the quotient are off on average, 3.9e-4 of the result in the mean
    square.  Sums that keep 13 bits are 22e-4 off."""
    g = torch.Generator().manual_seed(rows)
    x = (torch.randn(rows, D, generator=g, dtype=torch.float64)).to(torch.float16).double()
    w = {n: torch.randn(*s, generator=g, dtype=torch.float64).mul_(s[1] ** -0.5).to(torch.float16).double()
         for n, s in (("gate", (H, D)), ("up", (H, D)), ("down", (D, H)))}
    b = {n: torch.randn(v.shape[0], generator=g, dtype=torch.float64).mul_(0.1).float().double() for n, v in w.items()}
    def eight(t, square):
        q, s = F.quantize(t, square)
        return q * F.expand(s, *t.shape, square)
    x8, w8 = eight(x, False), {n: eight(v, True) for n, v in w.items()}
    layer = layer_of(w, b, "f16")
    b = {n: v.to(torch.float16).double() for n, v in b.items()}  # as the layer's weights are held
    gate, up = x8 @ w8["gate"].T + b["gate"], x8 @ w8["up"].T + b["up"]
    want = eight(gate / (1 + torch.exp(-gate)) * up, False) @ w8["down"].T + b["down"]
    got = layer.forward_fp8(x.to(torch.float16).cuda()).cpu().double()
    assert (got - want).norm() / want.norm() < (2.0 ** -22 + 3.9e-4 ** 2) ** 0.5
