"""An MoE layer's experts under the caller's routing (MoeLayer.forward_routed),
alone and in the chain that a block runs: norm/modulate, logits, route,
experts, block seam.

Bars: those of the layer's own forward against the oracle (tests/_gpu.py).
Where the layer's own router chose, the bits have to be the same.
"""
import numpy as np
import pytest
import torch

import nomas_moe as nm
import oracle as O
from _common import rounded, small_case
from _gpu import TOL, layer_from_tensors, rel_err, to_device

pytestmark = pytest.mark.gpu


def case(rows, D, E, k, H, dtype, seed, s=0.0):
    t, x = small_case(rows, D, E, k, H, seed, dense=s > 0, router_std=0.1)
    layer = layer_from_tensors(t, dtype, D, H, E, k, s)
    rt, xm = rounded(t, x, dtype)
    p, dense = nm.workloads.oracle_params(rt, E)
    return layer, to_device(x, dtype), xm, p, dense


def plain(xm, p, idx, w, s=0.0, dense=None):
    """sum_j w_j FFN_idx_j(x) in f64 (an index outside 0..E-1 adds nothing)."""
    x = xm.astype(np.float64)

    def ffn(q):
        g = x @ q[0].T.astype(np.float64) + q[1]
        u = x @ q[2].T.astype(np.float64) + q[3]
        return (g / (1 + np.exp(-g)) * u) @ q[4].T.astype(np.float64) + q[5]

    E = p["wr"].shape[0]
    y = np.zeros_like(x)
    for e in range(E):
        gate = np.where(idx == e, w.astype(np.float64), 0).sum(1)
        if gate.any():
            y += gate[:, None] * ffn([p[n][e] for n in ("wg", "bg", "wu", "bu", "wd", "bd")])
    if s > 0:
        y += s * ffn([dense[n] for n in ("wg", "bg", "wu", "bu", "wd", "bd")])
    return y


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,D,E,k,H,s", [
    (1, 64, 4, 2, 96, 0.0), (64, 256, 8, 2, 128, 0.0), (333, 192, 6, 3, 100, 0.5), (700, 256, 16, 4, 256, 0.0),
])
def test_the_routers_own_routing_gives_its_bits(dtype, rows, D, E, k, H, s):
    layer, x, *_ = case(rows, D, E, k, H, dtype, 40 + rows, s)
    want = layer.forward(x)
    idx, w, counts, _ = layer.routing(rows)
    got = layer.forward_routed(x, torch.from_numpy(idx).cuda(), torch.from_numpy(w).cuda())
    assert torch.equal(got, want)
    i2, w2, c2, gap = layer.routing(rows)
    assert np.array_equal(i2, idx) and np.array_equal(w2, w) and np.array_equal(c2, counts)
    assert np.isposinf(gap).all()
    # slots in any order
    perm = np.random.default_rng(1).permuted(np.tile(np.arange(k), (rows, 1)), axis=1)
    got = layer.forward_routed(x, torch.from_numpy(np.take_along_axis(idx, perm, 1)).cuda(),
                               torch.from_numpy(np.take_along_axis(w, perm, 1)).cuda())
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("s", [0.0, 0.5])
def test_empty_slots_and_repeated_experts(dtype, s):
    rows, D, E, k, H = 217, 128, 8, 3, 160
    layer, x, xm, p, dense = case(rows, D, E, k, H, dtype, 51, s)
    g = np.random.default_rng(52)
    idx = g.permuted(np.tile(np.arange(E), (rows, 1)), axis=1)[:, :k].astype(np.int32)
    w = g.random((rows, k)).astype(np.float32)
    idx[g.random((rows, k)) < 0.3] = -1
    idx[5] = -1                                   # nothing is left
    idx[64:128] = -1                              # a whole chunk of rows
    idx[6] = [3, 3, 3]                            # one expert, three times
    idx[7] = [2, -1, 2]
    idx[8] = [E, 2 ** 31 - 1, -2 ** 31]           # no experts
    got = layer.forward_routed(x, torch.from_numpy(idx).cuda(), torch.from_numpy(w).cuda())
    want = plain(xm, p, idx, w, s, dense)
    assert rel_err(got.float().cpu().numpy(), want) <= TOL[dtype]
    if s == 0:
        assert (got[5] == 0).all() and (got[64:128] == 0).all() and (got[8] == 0).all()
    i2, w2, counts, _ = layer.routing(rows)
    assert (i2[5] == -1).all() and i2[6].tolist() == [3, -1, -1]
    assert w2[6, 0] == np.float32(np.float32(w[6, 0] + w[6, 1]) + w[6, 2])
    live = [set(r[(r >= 0) & (r < E)]) for r in idx]
    assert counts.tolist() == [sum(e in q for q in live) for e in range(E)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_no_row_has_an_expert(dtype):
    # (twice: what an earlier forward left in the buffers must not show, not even a NaN)
    rows, D = 130, 64
    layer, x, *_ = case(rows, D, 4, 2, 96, dtype, 55)
    layer.forward(torch.full_like(x, float("nan")))
    none = torch.full((rows, 2), -1, dtype=torch.int32, device="cuda")
    got = layer.forward_routed(x, none, torch.ones(rows, 2, device="cuda"))
    assert (got == 0).all()


def test_a_wide_output_past_the_last_level_cache():
    # the down GEMM's nontemporal output and the combine of whole rows
    rows, D, E, k, H = 26_000, 1536, 4, 4, 64
    layer, x, xm, p, _ = case(rows, D, E, k, H, "bf16", 57)
    g = np.random.default_rng(58)
    idx = np.tile(np.arange(E, dtype=np.int32), (rows, 1))
    idx[g.random((rows, k)) < 0.05] = -1
    assert rows * k * D * 2 > 256 << 20
    w = g.random((rows, k)).astype(np.float32)
    got = layer.forward_routed(x, torch.from_numpy(idx).cuda(), torch.from_numpy(w).cuda())
    sel = g.choice(rows, 200, replace=False)
    want = plain(xm[sel], p, idx[sel], w[sel])
    assert rel_err(got.float().cpu().numpy()[sel], want) <= TOL["bf16"]


@pytest.mark.parametrize("k", [20, 136])  # 136: the most that 256 experts allow
def test_many_experts_and_slots(k):
    rows, D, E, H = 150, 64, 256, 32
    layer, x, xm, p, _ = case(rows, D, E, k, H, "bf16", 59)
    g = np.random.default_rng(60)
    idx = g.permuted(np.tile(np.arange(E), (rows, 1)), axis=1)[:, :k].astype(np.int32)
    idx[g.random((rows, k)) < 0.1] = -1
    w = g.random((rows, k)).astype(np.float32)
    got = layer.forward_routed(x, torch.from_numpy(idx).cuda(), torch.from_numpy(w).cuda())
    assert rel_err(got.float().cpu().numpy(), plain(xm, p, idx, w)) <= TOL["bf16"]


def test_zero_rows_and_alternating_calls():
    layer, x, *_ = case(200, 64, 4, 2, 96, "bf16", 61)
    assert layer.forward_routed(x[:0], torch.empty(0, 2, dtype=torch.int32, device="cuda"),
                                torch.empty(0, 2, device="cuda")).shape == (0, 64)
    want = layer.forward(x)
    idx, w, _, _ = layer.routing(200)
    idx, w = torch.from_numpy(idx).cuda(), torch.from_numpy(w).cuda()
    for _ in range(3):  # (the split counters and empty-slot marks of one call do not reach the next)
        none = torch.full_like(idx, -1)
        assert (layer.forward_routed(x, none, w) == 0).all()
        assert torch.equal(layer.forward(x), want)
        assert torch.equal(layer.forward_routed(x, idx, w), want)


def test_chain_of_a_block_eager_and_captured():
    """norm_modulate -> logits -> route -> forward_routed -> block_seam, as a block runs them,
    against the same chain in f64; then captured, replayed with other inputs."""
    B, S, D, E, k, H, dtype = 2, 150, 128, 8, 2, 192, "bf16"
    layer, x, *_ = case(B * S, D, E, k, H, dtype, 63)
    t, _ = small_case(B * S, D, E, k, H, 63, router_std=0.1)
    rt, _ = rounded(t, np.zeros((1, 1), np.float32), dtype)
    p, _ = nm.workloads.oracle_params(rt, E)
    x = x.view(B, S, D)
    g = torch.Generator(device="cuda").manual_seed(64)
    sh, sc, gt, sh2, sc2 = (0.3 * torch.randn(B, D, generator=g, device="cuda") for _ in range(5))
    wr = torch.from_numpy(p["wr"]).cuda()
    post = 1 + 0.1 * torch.randn(D, generator=g, device="cuda")
    bias = 0.02 * torch.randn(E, generator=g, device="cuda")

    def chain():
        h = nm.norm_modulate(x, sh, sc)
        logits = h.float() @ wr.T
        idx, w, counts = nm.route(logits, k, scoring="sigmoid", bias=bias, groups=4, top_groups=2, scale=1.5)
        y = layer.forward_routed(h, idx, w)
        out, h2 = nm.block_seam(x, y, gt, sh2, sc2, post_norm=True, post_w=post, residual_scale=0.7)
        return h, logits, idx, w, counts, y, out, h2

    h, logits, idx, w, counts, y, out, h2 = chain()
    torch.cuda.synchronize()
    import _block_ops as ref
    i, v, c = ref.route(logits.double().cpu().numpy().reshape(-1, E), k, "sigmoid", bias.double().cpu().numpy(), 4,
                        2, 2, True, 1.5)
    assert np.array_equal(idx.cpu().numpy().reshape(-1, k), i) and np.array_equal(counts.cpu().numpy(), c)
    want = plain(h.float().cpu().numpy().reshape(-1, D), p, i, v)
    assert rel_err(y.float().cpu().numpy().reshape(-1, D), want) <= TOL[dtype]
    o, eo, n, en = ref.seam_errors(*(q.double().cpu() for q in (x, y, gt, sh2, sc2)), True, post.double().cpu(),
                                   None, 0.7, 1e-6, dtype)
    assert ((out.double().cpu() - o).abs() <= eo).all() and ((h2.double().cpu() - n).abs() <= en).all()

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        chain()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            got = chain()
    keep = x.clone()
    for r in range(4):
        x.copy_(keep * (1 + r))
        graph.replay()
        torch.cuda.synchronize()
        eager = chain()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager)), r


def test_refusals_with_a_layer():
    layer, x, *_ = case(40, 64, 4, 2, 96, "bf16", 71)
    i = torch.zeros(40, 2, dtype=torch.int32, device="cuda")
    w = torch.ones(40, 2, device="cuda")
    L, p = nm._lib.lib(), x.data_ptr()
    y = torch.empty_like(x)
    for args in ((p, None, w.data_ptr()), (p, i.data_ptr(), None), (None, i.data_ptr(), w.data_ptr()),
                 (p + 2, i.data_ptr(), w.data_ptr()), (p, i.data_ptr() + 2, w.data_ptr())):
        assert L.nomas_moe_forward_routed(layer._h, *args, y.data_ptr(), 40, None) == 2
    assert L.nomas_moe_forward_routed(layer._h, p, i.data_ptr(), w.data_ptr(), y.data_ptr(), -1, None) == 2
    for bad in ((x, i.long(), w), (x, i, w.half()), (x, i[:, :1], w), (x, i, w[:20]), (x, i.cpu(), w), (x.float(), i, w)):
        with pytest.raises(nm.NomasError):
            layer.forward_routed(*bad)


def test_streams_are_ordered():
    # forwards of one handle on different streams share its workspace and wait for each other
    layer, x, *_ = case(900, 128, 8, 2, 192, "bf16", 73)
    want = layer.forward(x)
    idx, w, _, _ = layer.routing(900)
    idx, w = torch.from_numpy(idx).cuda(), torch.from_numpy(w).cuda()
    flip = layer.forward_routed(x, idx.flip(0), w)
    torch.cuda.synchronize()
    s = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(6):
        with torch.cuda.stream(s[0]):
            a = layer.forward_routed(x, idx, w)
        with torch.cuda.stream(s[1]):
            b = layer.forward_routed(x, idx.flip(0), w)
        c = layer.forward(x)
        torch.cuda.synchronize()
        assert torch.equal(a, want) and torch.equal(b, flip) and torch.equal(c, want)
