"""The MoE layer on few rows (MoeLayer.forward_few) against its definition in 64 bits.

The bounds count the roundings: sums of n terms in f32 are off by at most n steps of 2^-24 of
the terms' magnitudes (the matrix cores may truncate: a step, not half of one), the hidden
activations are rounded to the model dtype (half a step), and y once more.
"""
import numpy as np
import pytest
import torch

import nomas_moe as nm
import _fp8 as F
from _common import rounded, small_case
from _gpu import layer_from_tensors, to_device

pytestmark = pytest.mark.gpu

U = 2.0 ** -23
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
TINY = {"f32": 0.0, "bf16": 0.0, "f16": 2.0 ** -25}


def case(rows, D, E, k, H, dtype, seed, s=0.0, fp8=False):
    t, x = small_case(rows, D, E, k, H, seed, dense=s > 0, router_std=0.1)
    layer = layer_from_tensors(t, dtype, D, H, E, k, s)
    rt, xm = rounded(t, x, dtype)
    p, dense = nm.workloads.oracle_params(rt, E)
    layer.wr = p["wr"]
    names = ("wg", "bg", "wu", "bu", "wd", "bd")
    ffn = [[np.asarray(p[n][e], np.float64) for n in names] for e in range(E)]
    ffn += [[np.asarray(dense[n], np.float64) for n in names]] if s > 0 else []
    if fp8:
        layer.quantize()
        for f in ffn:
            for i in (0, 2, 4):
                q, c = F.quantize(torch.from_numpy(f[i]), True)
                f[i] = (q * F.expand(c, *q.shape, True)).numpy()
    return layer, to_device(x, dtype), xm, ffn


def plain(xm, ffn, idx, w, dtype, s=0.0):
    """(y, bound) in f64 (an index outside 0 .. E - 1 adds nothing)."""
    x = xm.astype(np.float64)
    E = len(ffn) - (1 if s > 0 else 0)
    y, off = np.zeros_like(x), np.zeros_like(x)
    for e, (wg, bg, wu, bu, wd, bd) in enumerate(ffn):
        gate = np.where(idx == e, w.astype(np.float64), 0).sum(1) if e < E else np.full(len(x), s)
        if not gate.any():
            continue
        D, H = x.shape[1], wg.shape[0]
        g, u = x @ wg.T + bg, x @ wu.T + bu
        eg = (D + 16) * U * (np.abs(x) @ np.abs(wg).T + np.abs(bg))
        eu = (D + 16) * U * (np.abs(x) @ np.abs(wu).T + np.abs(bu))
        sig = 1 / (1 + np.exp(-g))
        h = g * sig * u
        # silu' is at most 1.1; exp's argument, its own error, the reciprocal and two products
        eh = 1.1 * eg * (np.abs(u) + eu) + np.abs(g * sig) * eu + (np.abs(g) + 8) * U * np.abs(h)
        eh += HALF[dtype] * (np.abs(h) + eh) + TINY[dtype]
        o = h @ wd.T + bd
        eo = eh @ np.abs(wd).T + (H + 16) * U * ((np.abs(h) + eh) @ np.abs(wd).T + np.abs(bd))
        y += gate[:, None] * o
        off += np.abs(gate)[:, None] * (eo + (len(ffn) + 16) * U * np.abs(o))
    return y, off + HALF[dtype] * (np.abs(y) + off) + TINY[dtype]


def near(got, want, off):
    assert np.all(np.abs(got.double().cpu().numpy() - want) <= off)


SHAPES = [  # rows, dim, experts, top_k, hidden, shared dense
    (1, 8, 1, 1, 1, 0.0), (1, 64, 4, 2, 96, 0.0), (2, 64, 4, 2, 128, 0.5), (5, 136, 8, 3, 100, 0.0), (16, 256, 16, 4, 72, 0.25),
    (17, 200, 3, 2, 333, 0.0), (32, 512, 8, 2, 256, 0.0), (33, 1000, 5, 5, 130, 0.7), (64, 1032, 2, 1, 520, 0.0),
    (64, 72, 256, 8, 40, 0.5), (7, 2304, 64, 6, 264, 0.0), (3, 264, 256, 64, 24, 0.5), (64, 40, 64, 64, 24, 0.0),
]


@pytest.mark.parametrize("dtype,fp8", [("f32", False), ("bf16", False), ("f16", False), ("bf16", True), ("f16", True)])
@pytest.mark.parametrize("rows,D,E,k,H,s", SHAPES)
def test_the_routers_choice(rows, D, E, k, H, s, dtype, fp8):
    layer, x, xm, ffn = case(rows, D, E, k, H, dtype, 100 + rows + D, s, fp8)
    big = torch.full((rows * D + 64,), 7.0, dtype=x.dtype, device="cuda")
    y = layer.forward_few(x, fp8=fp8, out=big[:rows * D].view(rows, D))
    idx, w, counts, gap = layer.routing(rows)
    near(y, *plain(xm, ffn, idx, w, dtype, s))
    assert bool((big[rows * D:] == 7.0).all())
    # The layer's own router: of 16-bit products both sum 32 at a time in f32 (at most 32 steps of 2^-23 of their
    # magnitudes; f32 inputs are summed in f64) and those sums in f64, in another order.  So two logits
    # are that far apart twice; a weight is a ratio of exponentials of differences of logits, each exponential
    # with an f32 argument and its own error.
    layer.forward(x)
    i2, w2, c2, g2 = layer.routing(rows)
    dl = 2 * 32 * U * (np.abs(xm.astype(np.float64)) @ np.abs(layer.wr.astype(np.float64)).T).max(1)
    dl = dl if dtype != "f32" else 2.0 ** -40 + 0 * dl
    sure = (gap > dl) | np.isinf(gap)
    assert sure.any() and np.array_equal(idx[sure], i2[sure]) and counts.sum() == rows * k
    spread = 64.0  # (no logit here is further from the largest)
    rel = np.expm1(2 * dl) + 4 * (spread + 4) * U
    assert np.all(np.abs(w - w2)[sure] <= (rel[:, None] * np.abs(w2))[sure])
    both = sure & np.isfinite(gap)
    assert np.all(np.abs(gap[both] - g2[both]) <= 2 * dl[both] + U * np.abs(g2[both])) and np.array_equal(np.isinf(gap), np.isinf(g2))
    if sure.all():
        assert np.array_equal(counts, c2)


@pytest.mark.parametrize("dtype,fp8", [("f32", False), ("bf16", False), ("f16", True)])
@pytest.mark.parametrize("rows,D,E,k,H,s", [s for s in SHAPES if s[3] < 64])
def test_the_callers_routing(rows, D, E, k, H, s, dtype, fp8):
    layer, x, xm, ffn = case(rows, D, E, k, H, dtype, 300 + rows + D, s, fp8)
    r = np.random.default_rng(rows)
    idx = r.integers(-2, E + 1, (rows, k)).astype(np.int32)  # empty slots, repeated experts, any order
    w = r.normal(size=(rows, k)).astype(np.float32)
    idx[rows // 2] = -1  # a row with nothing
    w[idx < 0] = np.nan  # what stands beside an empty slot is not used
    w[idx >= E] = np.inf
    used = np.where((idx >= 0) & (idx < E), w, 0)
    y = layer.forward_few(x, torch.from_numpy(idx).cuda(), torch.from_numpy(w).cuda(), fp8=fp8)
    near(y, *plain(xm, ffn, np.where(idx < E, idx, -1), used, dtype, s))
    if s == 0.0:
        assert not y[rows // 2].any()
    with pytest.raises(nm.NomasError, match="caller's routing"):
        layer.routing(rows)


@pytest.mark.parametrize("rows", [2, 40])
@pytest.mark.parametrize("E,k", [(4, 1), (16, 3), (64, 8), (64, 64), (200, 6), (256, 1)])
def test_ties_and_near_ties(rows, E, k):
    """Equal logits: the lowest index; logits that differ by 2^-40 only, or by f32's last bit: the larger one."""
    D, H = 64, 16
    t, _ = small_case(rows, D, E, k, H, 11)
    r = np.random.default_rng(E + k)
    fine = r.permutation(E)
    fine[: E // 2] = fine[0]  # half of them equal
    wr = np.zeros((E, D), np.float32)
    wr[:, 0], wr[:, 1], wr[:, 2] = 1.0, fine * 2.0 ** -20, r.integers(0, 2, E) * 2.0 ** -23
    t["blocks.0.moe.router.weight"] = wr
    layer = layer_from_tensors(t, "f32", D, H, E, k, 0.0)
    x = np.zeros((rows, D), np.float32)
    x[:, 0] = 1.0
    x[:, 1] = 2.0 ** -20
    x[1::2, 2] = 1.0
    layer.forward_few(torch.from_numpy(x).cuda())
    logits = x.astype(np.float64) @ wr.astype(np.float64).T
    idx, w, counts, gap = layer.routing(rows)
    for i in range(rows):
        order = sorted(range(E), key=lambda e: (-logits[i, e], e))
        assert list(idx[i]) == sorted(order[:k])
        p = np.exp(logits[i] - logits[i].max())[idx[i]]
        assert np.allclose(w[i], p / (p.sum() + 1e-9 * p.sum()), rtol=1e-6, atol=0)
        assert gap[i] == (np.inf if k == E else np.float32(logits[i, order[k - 1]] - logits[i, order[k]]))


@pytest.mark.parametrize("fp8", [False, True])
def test_rows_do_not_touch_each_other(fp8):
    layer, x, _, _ = case(20, 264, 6, 2, 200, "bf16", 7, fp8=fp8)
    layer.forward(x)
    idx, w, _, _ = layer.routing(20)
    idx, w = torch.from_numpy(idx).cuda(), torch.from_numpy(w).cuda()
    want = layer.forward_few(x, idx, w, fp8=fp8)
    x[3], x[11, 5], x[19, 263] = float("nan"), float("inf"), float("-inf")
    got = layer.forward_few(x, idx, w, fp8=fp8)
    ok = torch.ones(20, dtype=torch.bool, device="cuda")
    ok[[3, 11, 19]] = False
    assert torch.equal(got[ok], want[ok])
    assert bool(got[3].isnan().all()) and not bool(got[11].isfinite().all()) and not bool(got[19].isfinite().all())


@pytest.mark.parametrize("dtype,fp8", [("bf16", False), ("bf16", True), ("f32", False)])
def test_calls_in_a_row(dtype, fp8):
    """The same bits again, in place, with leading dimensions, strides and other row counts between."""
    layer, x, _, _ = case(48, 512, 16, 4, 384, dtype, 5, 0.3, fp8)
    want = layer.forward_few(x, fp8=fp8)
    for n in (1, 16, 31, 48):
        assert torch.equal(layer.forward_few(x[:n], fp8=fp8), layer.forward_few(x[:n], fp8=fp8))
    for _ in range(20):
        assert torch.equal(layer.forward_few(x, fp8=fp8), want)
    assert torch.equal(layer.forward_few(x.view(2, 24, 512), fp8=fp8), want.view(2, 24, 512))
    assert torch.equal(layer.forward_few(x.T.contiguous().T, fp8=fp8), want)
    layer.forward(x)
    y = x.clone()
    assert torch.equal(layer.forward_few(y, fp8=fp8, out=y), want) and torch.equal(y, want)
    assert layer.forward_few(x[:0], fp8=fp8).shape == (0, 512)


def test_the_other_forwards_stay():
    layer, x, _, _ = case(70, 256, 8, 2, 128, "bf16", 3)
    want = layer.forward(x)
    layer.quantize()
    layer.quantize()
    layer.forward_few(x[:9], fp8=True)
    assert torch.equal(layer.forward(x), want)


@pytest.mark.parametrize("fp8", [False, True])
def test_streams_order_and_capture(fp8):
    layer, x, _, _ = case(12, 512, 8, 2, 768, "bf16", 8, fp8=fp8)
    other = torch.randn_like(x)
    want, want2 = layer.forward_few(x, fp8=fp8), layer.forward_few(other, fp8=fp8)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (s1, s2):
        s.wait_stream(torch.cuda.current_stream())
    outs = []
    for _ in range(10):  # calls on two streams share the workspace: they wait for each other
        with torch.cuda.stream(s1):
            outs.append((layer.forward_few(x, fp8=fp8), want))
        with torch.cuda.stream(s2):
            outs.append((layer.forward_few(other, fp8=fp8), want2))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in outs)
    g = torch.cuda.CUDAGraph()
    cap = torch.cuda.Stream()
    cap.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(cap):
        layer.forward_few(x, fp8=fp8)
    torch.cuda.current_stream().wait_stream(cap)
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=cap):
        y = layer.forward_few(x, fp8=fp8)
    for seed in range(4):
        x.copy_(torch.randn(12, 512, generator=torch.Generator().manual_seed(seed)))
        eager = layer.forward_few(x, fp8=fp8)
        layer.forward_few(torch.randn(64, 512, device="cuda", dtype=torch.bfloat16), fp8=fp8)  # more rows between
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, eager)


def test_states_refused():
    layer, x, _, _ = case(4, 64, 4, 2, 96, "bf16", 1)
    idx, w = torch.zeros(4, 2, dtype=torch.int32, device="cuda"), torch.ones(4, 2, device="cuda")
    with pytest.raises(nm.NomasError, match="quantize it first"):
        layer.forward_few(x, fp8=True)
    with pytest.raises(nm.NomasError, match="up to 64"):
        layer.forward_few(torch.zeros(65, 64, dtype=torch.bfloat16, device="cuda"))
    for kw in (dict(idx=idx), dict(w=w)):
        with pytest.raises(nm.NomasError, match="both be given"):
            layer.forward_few(x, **kw)
    with pytest.raises(nm.NomasError, match="^idx"):
        layer.forward_few(x, idx.long(), w)
    with pytest.raises(nm.NomasError, match="^w"):
        layer.forward_few(x, idx, w[:, :1])
    with pytest.raises(nm.NomasError, match="dtype"):
        layer.forward_few(x.float())
    with pytest.raises(nm.NomasError, match="last dim"):
        layer.forward_few(x[:, :32])
    with pytest.raises(nm.NomasError, match="GPU"):
        layer.forward_few(x.cpu())
    both = torch.zeros(4 * 64 * 2 + 64, dtype=torch.uint8, device="cuda")
    y, i = both[:512].view(torch.bfloat16).view(4, 64), both[480:512].view(torch.int32).view(4, 2)
    with pytest.raises(nm.NomasError, match="shares"):
        layer.forward_few(x, i, w, out=y)
    f32, *_ = case(4, 64, 4, 2, 96, "f32", 1)
    with pytest.raises(nm.InvalidConfig, match="f32"):
        f32.quantize()


@pytest.mark.parametrize("fp8", [False, True])
def test_graphs_that_share_a_workspace_and_layers_side_by_side(fp8):
    """Two graphs of one layer, of few and of many rows, replayed in turn, while another layer runs on another stream."""
    layer, x, _, _ = case(64, 512, 8, 2, 768, "bf16", 9, fp8=fp8)
    beside, xb, _, _ = case(20, 256, 16, 3, 200, "bf16", 10, fp8=fp8)
    want = {n: layer.forward_few(x[:n], fp8=fp8) for n in (3, 64)}
    wb = beside.forward_few(xb, fp8=fp8)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    graphs = {}
    for n in want:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            y = layer.forward_few(x[:n], fp8=fp8)
        graphs[n] = g, y
    outs = []
    for _ in range(4):
        for n in (64, 3, 3):
            g, y = graphs[n]
            with torch.cuda.stream(s):
                y.zero_()
                g.replay()
                outs.append((y.clone(), want[n]))
            outs.append((beside.forward_few(xb, fp8=fp8), wb))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in outs)
