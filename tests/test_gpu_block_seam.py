"""The seam between two branches of a block (nm.block_seam) and its gradients on
the GPU, against their formulas in 64 bits, with bounds on the errors that the
f32 evaluation and the outputs' types allow (tests/_block_ops.py)."""
from concurrent.futures import ThreadPoolExecutor

import numpy as np
import pytest
import torch

import nomas_moe as nm
import _block_ops as ref

pytestmark = pytest.mark.gpu

EPS = 1e-6


def inputs(B, S, D, dtype, seed, names=("x", "y")):
    g = torch.Generator().manual_seed(seed)
    t = {n: (torch.randn(B, S, D, generator=g) * torch.exp(0.5 * torch.randn(B, S, 1, generator=g)))
         .to(ref.TORCH[dtype]) for n in names}
    for n in ("gate", "shift", "scale"):
        t[n] = 0.5 * torch.randn(B, D, generator=g)
    for n in ("norm_w", "post_w"):
        t[n] = 1 + 0.3 * torch.randn(D, generator=g)
    return t


def dev(t):
    return None if t is None else t.cuda()


def wide(t):
    return None if t is None else t.double()


def check(t, dtype, post, alpha, drop=()):
    t = {k: None if k in drop else v for k, v in t.items()}
    pw = t["post_w"] if post else None
    out, h = nm.block_seam(dev(t["x"]), dev(t["y"]), dev(t["gate"]), dev(t["shift"]), dev(t["scale"]),
                           post_norm=post, post_w=dev(pw), norm_w=dev(t["norm_w"]), residual_scale=alpha, eps=EPS)
    torch.cuda.synchronize()
    o, eo, n, en = ref.seam_errors(wide(t["x"]), wide(t["y"]), wide(t["gate"]), wide(t["shift"]), wide(t["scale"]),
                                   post, wide(pw), wide(t["norm_w"]), alpha, EPS, dtype)
    assert ((out.double().cpu() - o).abs() <= eo).all(), (out.double().cpu() - o).abs().max()
    assert ((h.double().cpu() - n).abs() <= en).all(), (h.double().cpu() - n).abs().max()
    return out, h


SHAPES = [
    (1, 1, 8), (1, 3, 16), (5, 1, 64), (2, 150, 256), (3, 7, 264), (1, 70, 1000), (4, 33, 512),
    (2, 19, 520), (1, 40, 2048), (7, 2, 1032), (1, 9, 4104), (2, 5, 8192), (1, 3, 8200), (1, 2, 16384), (300, 1, 128),
    (2, 700, 64), (1, 13, 16384), (2, 9, 12296), (5, 60, 768), (6, 100, 1536),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("B,S,D", SHAPES)
def test_forward(dtype, B, S, D):
    t = inputs(B, S, D, dtype, D + S)
    check(t, dtype, True, 1.0)
    check(t, dtype, False, 0.5)


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("drop", [("gate",), ("shift",), ("scale",), ("norm_w",), ("post_w",),
                                  ("gate", "shift", "scale", "norm_w", "post_w")])
def test_parameters_left_out(post, drop):
    check(inputs(2, 37, 136, "bf16", 3), "bf16", post, 1.0, drop)


@pytest.mark.parametrize("D", [72, 1536])
def test_without_the_second_norm_and_in_place(D):
    t = {k: dev(v) for k, v in inputs(2, 45, D, "bf16", 5).items()}
    kw = dict(post_norm=True, post_w=t["post_w"], residual_scale=0.5)
    want, h = nm.block_seam(t["x"], t["y"], t["gate"], t["shift"], t["scale"], norm_w=t["norm_w"], **kw)
    out, none = nm.block_seam(t["x"], t["y"], t["gate"], norm=False, **kw)
    assert none is None and torch.equal(out, want)
    for first, second in (("x", "y"), ("y", "x")):
        u = {n: t[n].clone() for n in ("x", "y")}
        o, n = nm.block_seam(u["x"], u["y"], t["gate"], t["shift"], t["scale"], norm_w=t["norm_w"], out=u[first],
                             h=u[second], **kw)
        assert o is u[first] and torch.equal(o, want) and torch.equal(n, h)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rows_of_zeros_and_of_extremes(dtype):
    t = inputs(1, 8, 96, dtype, 7)
    t["x"][0, 0] = 0
    t["y"][0, 0] = 0          # out and its norm: zero, h: shift
    t["y"][0, 1] = 1e-18      # far below eps
    t["x"][0, 2] *= 1e4
    out, h = check(t, dtype, True, 1.0)
    assert (out[0, 0] == 0).all() and torch.equal(h[0, 0].cpu(), t["shift"][0].to(h.dtype))
    t["x"][0, 3, 5] = float("nan")
    t["y"][0, 4, 7] = float("inf")
    out, h = nm.block_seam(dev(t["x"]), dev(t["y"]), dev(t["gate"]), dev(t["shift"]), dev(t["scale"]))
    assert torch.isnan(h[0, 3]).all() and torch.isfinite(h[0, [0, 1, 2, 5, 6, 7]]).all()
    assert torch.isfinite(out[0, 4, :7]).all() and not torch.isfinite(out[0, 4, 7])


def test_rows_past_4_gib():
    # 2^31 elements and more: the last rows' offsets pass 32 bits in elements and bytes
    B, S, D = 1, 270_000, 8192
    x = torch.zeros(B, S, D, dtype=torch.bfloat16, device="cuda")
    y = torch.zeros(B, S, D, dtype=torch.bfloat16, device="cuda")
    t = inputs(1, 3, D, "bf16", 11)
    x[:, -3:], y[:, -3:] = t["x"].cuda(), t["y"].cuda()
    p = {k: dev(t[k]) for k in ("gate", "shift", "scale")}
    out, h = nm.block_seam(x, y, p["gate"], p["shift"], p["scale"], post_norm=True, out=x, h=y)
    o, n = nm.block_seam(t["x"].cuda(), t["y"].cuda(), p["gate"], p["shift"], p["scale"], post_norm=True)
    assert torch.equal(out[:, -3:], o) and torch.equal(h[:, -3:], n)
    assert (out[:, :-3] == 0).all()


# ---- gradients --------------------------------------------------------------------

def check_grad(t, dtype, post, alpha, drop=()):
    t = {k: None if k in drop else v for k, v in t.items()}
    pw = t["post_w"] if post else None
    got = nm.block_seam_backward(dev(t["dout"]), dev(t["dh"]), dev(t["out"]), dev(t["y"]), dev(t["gate"]),
                                 dev(t["scale"]), post_norm=post, post_w=dev(pw), norm_w=dev(t["norm_w"]),
                                 residual_scale=alpha, eps=EPS)
    torch.cuda.synchronize()
    want, mag = ref.seam_grad(*(wide(t[n]) for n in ("dout", "dh", "out", "y", "gate", "scale")), post, wide(pw),
                              wide(t["norm_w"]), alpha, EPS)
    assert sorted(got) == sorted(want)
    some = t["dout"] if t["dout"] is not None else t["dh"]
    rows = some.shape[0] * some.shape[1]
    for n, w in want.items():
        g = got[n].double().cpu()
        assert g.shape == w.shape and got[n].dtype == (some.dtype if n in ("dx", "dy") else torch.float32)
        off = (g - w).abs() - ref.seam_grad_bound(n, w, mag[n], rows, dtype)
        assert (off <= 0).all(), (n, off.max())
    return got


NAMES = ("dout", "dh", "out", "y")


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("B,S,D", SHAPES)
def test_gradients(dtype, B, S, D):
    t = inputs(B, S, D, dtype, 2 * D + S, NAMES)
    check_grad(t, dtype, True, 1.0)
    check_grad(t, dtype, False, 0.5)


@pytest.mark.parametrize("drop", [(), ("scale", "norm_w"), ("gate", "post_w")])
@pytest.mark.parametrize("B,S,D", [(4, 40, 1032), (13, 40, 1032), (64, 16, 1536), (9, 300, 72), (17, 120, 264)])
def test_gradients_of_many_sequences(drop, B, S, D):
    check_grad(inputs(B, S, D, "f32", 17, NAMES), "f32", True, 1.0, drop)


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("B,S,D", [(2, 37, 136), (3, 300, 512), (40, 3, 1032)])
@pytest.mark.parametrize("drop", [("gate",), ("scale",), ("norm_w",), ("post_w",), ("dout",),
                                  ("dh", "out", "scale", "norm_w"), ("gate", "scale", "norm_w", "post_w", "dout")])
def test_gradients_with_parts_left_out(post, drop, B, S, D):
    check_grad(inputs(B, S, D, "bf16", 13, NAMES), "bf16", post, 1.0, drop)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_gradients_without_a_branch(dtype):
    # those of norm_modulate
    for B, S, D in ((2, 37, 136), (30, 1, 264)):
        check_grad(inputs(B, S, D, dtype, 15, NAMES), dtype, False, 1.0, ("y", "gate"))


def test_gradients_of_cancelled_rows():
    # dh along out: nothing of it is left but eps' share
    t = inputs(1, 6, 256, "f32", 17, NAMES)
    t["dh"] = t["out"].clone()
    t["scale"], t["norm_w"] = torch.zeros(1, 256), torch.ones(256)
    t["out"][0, 2] = 0
    t["dh"][0, 2] = 0
    check_grad(t, "f32", True, 1.0)


@pytest.mark.parametrize("post", [False, True])
def test_gradients_against_differences(post):
    B, S, D, alpha = 2, 5, 48, 0.6
    t = {k: v.double() for k, v in inputs(B, S, D, "f32", 19).items()}
    g = torch.Generator().manual_seed(20)
    dout, dh = (torch.randn(B, S, D, generator=g).double() for _ in range(2))
    pw = t["post_w"] if post else None

    def loss(p):
        o, h = ref.seam(p["x"], p["y"], p["gate"], p["shift"], p["scale"], post, p["post_w"] if post else None,
                        p["norm_w"], alpha, EPS)
        return float((o * dout).sum() + (h * dh).sum())

    out, _ = nm.block_seam(*(t[n].float().cuda() for n in ("x", "y", "gate", "shift", "scale")), post_norm=post,
                           post_w=dev(pw if pw is None else pw.float()), norm_w=t["norm_w"].float().cuda(),
                           residual_scale=alpha, eps=EPS)
    got = nm.block_seam_backward(dout.float().cuda(), dh.float().cuda(), out, t["y"].float().cuda(),
                                 t["gate"].float().cuda(), t["scale"].float().cuda(), post_norm=post,
                                 post_w=dev(pw if pw is None else pw.float()), norm_w=t["norm_w"].float().cuda(),
                                 residual_scale=alpha, eps=EPS)
    for n in ("x", "y", "gate", "shift", "scale", "norm_w") + (("post_w",) if post else ()):
        u = torch.randn(t[n].shape, generator=g).double()
        step = 1e-5
        diff = (loss({**t, n: t[n] + step * u}) - loss({**t, n: t[n] - step * u})) / (2 * step)
        d = got["d" + n].double().cpu()
        # f32 inputs and sums of some hundred terms: 1e-6 of their magnitudes; differences: step^2
        assert abs(float((d * u).sum()) - diff) <= 1e-7 + 4e-6 * float((d * u).abs().sum()), n


def test_same_bits_again_in_place_and_captured():
    B, S, D = 3, 333, 768
    t = {k: dev(v) for k, v in inputs(B, S, D, "bf16", 23, NAMES).items()}
    kw = dict(post_norm=True, post_w=t["post_w"], norm_w=t["norm_w"], residual_scale=0.5)

    def call():
        return nm.block_seam_backward(t["dout"], t["dh"], t["out"], t["y"], t["gate"], t["scale"], **kw)

    want = call()
    for k, v in call().items():
        assert torch.equal(v, want[k]), k
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            got = call()
    keep = t["dh"].clone()
    for r in range(4):
        t["dh"].copy_(keep * (r + 1))
        graph.replay()
        torch.cuda.synchronize()
        eager = call()
        torch.cuda.synchronize()
        for k in want:
            assert torch.equal(got[k], eager[k]), (r, k)
    t["dh"].copy_(keep)
    # dx over dh and dy over y, through the C call
    L = nm._lib.lib()
    need = L.nomas_block_seam_workspace(B * S, D, S)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    dg = torch.empty(B, D, device="cuda")
    rc = L.nomas_block_seam_backward(1, t["dout"].data_ptr(), t["dh"].data_ptr(), t["out"].data_ptr(),
                                     t["y"].data_ptr(), t["dh"].data_ptr(), t["y"].data_ptr(), B * S, D, S,
                                     t["gate"].data_ptr(), 1, t["post_w"].data_ptr(), 0.5, t["norm_w"].data_ptr(),
                                     t["scale"].data_ptr(), 1e-6, dg.data_ptr(), None, None, None, None,
                                     ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    assert torch.equal(t["dh"], want["dx"]) and torch.equal(t["y"], want["dy"]) and torch.equal(dg, want["dgate"])


def test_two_streams_at_once():
    t = [{k: dev(v) for k, v in inputs(2, 500, 640, "bf16", 40 + i, NAMES).items()} for i in range(2)]

    def call(u):
        o, h = nm.block_seam(u["dout"], u["y"], u["gate"], u["shift"], u["scale"], post_norm=True)
        g = nm.block_seam_backward(u["dout"], u["dh"], u["out"], u["y"], u["gate"], u["scale"], post_norm=True)
        return [o, h] + [g[k] for k in sorted(g)]

    want = [call(u) for u in t]
    torch.cuda.synchronize()
    s = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = []
        for u, st in zip(t, s):
            with torch.cuda.stream(st):
                got.append(call(u))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(got, want) for a, b in zip(x, y))


def test_two_host_threads():
    # wide rows of two widths: each call asks for its own share of LDS
    t = [{k: dev(v) for k, v in inputs(1, 9, D, "bf16", D, NAMES).items()} for D in (8192, 16384)]

    def call(u):
        g = nm.block_seam_backward(u["dout"], u["dh"], u["out"], u["y"], u["gate"], u["scale"], post_norm=True)
        return [g[k] for k in sorted(g)]

    want = [call(u) for u in t]
    torch.cuda.synchronize()
    with ThreadPoolExecutor(2) as pool:
        for _ in range(20):
            got = list(pool.map(call, t))
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for x, y in zip(got, want) for a, b in zip(x, y))


def test_strided_inputs_and_parameters_of_other_types():
    # the AdaLN chunks of one tensor, activations with a stride, 16-bit gains
    B, S, D = 2, 30, 96
    t = inputs(B, S, D, "bf16", 50)
    six = torch.cat([t["gate"], t["shift"], t["scale"]], 1).cuda()
    gate, shift, scale = six.chunk(3, 1)
    wide = torch.empty(B, S, 2 * D, dtype=torch.bfloat16, device="cuda")
    wide[..., :D], wide[..., D:] = t["x"].cuda(), t["y"].cuda()
    w16 = t["norm_w"].bfloat16().cuda()
    got = nm.block_seam(wide[..., :D], wide[..., D:], gate, shift, scale, norm_w=w16)
    want = nm.block_seam(t["x"].cuda(), t["y"].cuda(), t["gate"].cuda(), t["shift"].cuda(), t["scale"].cuda(),
                         norm_w=w16.float())
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_empty_batches():
    z = torch.empty(2, 0, 64, dtype=torch.bfloat16, device="cuda")
    out, h = nm.block_seam(z, z)
    assert out.shape == h.shape == (2, 0, 64)
    got = nm.block_seam_backward(z, z, z, z, post_norm=True)
    assert got["dx"].shape == (2, 0, 64)
    for n in ("dgate", "dshift", "dscale", "dnorm_w", "dpost_w"):
        assert (got[n] == 0).all(), n
