"""Routing to experts (nm.route) and its gradient on the GPU, against their
definitions in 64 bits (tests/_block_ops.py).

The choice and the counts have to be equal.  Weights: an exponential's relative
error is its argument's in half steps of f32, and the score's, the sum's (a tree over at most
1,024 experts) and the quotient's roundings come to 16 more.
"""
import numpy as np
import pytest
import torch

import nomas_moe as nm
import _block_ops as ref

pytestmark = pytest.mark.gpu


def logits_of(T, E, seed, dtype, std=1.0):
    g = np.random.default_rng(seed)
    l = torch.from_numpy((g.standard_normal((T, E)) * std + 0.5 * g.standard_normal(E)).astype(np.float32))
    return l.to(ref.TORCH[dtype])


def check(l, k, **kw):
    """Runs nm.route on the logits and compares it; returns (idx, w)."""
    b = kw.get("bias")
    idx, w, counts = nm.route(l.cuda(), k, **{**kw, "bias": None if b is None else b.cuda()})
    torch.cuda.synchronize()
    l64 = l.double().numpy().reshape(-1, l.shape[-1])
    want = ref.route(l64, k, **{**kw, "bias": None if b is None else b.double().numpy()})
    i, v = idx.cpu().numpy().reshape(-1, k), w.double().cpu().numpy().reshape(-1, k)
    assert idx.shape == w.shape == l.shape[:-1] + (k,)
    assert idx.dtype == torch.int32 and w.dtype == torch.float32
    bad = np.nonzero((i != want[0]).any(1))[0]
    assert not bad.size, f"{bad.size} rows differ, row {bad[0]}: {i[bad[0]]} for {want[0][bad[0]]}"
    assert np.array_equal(counts.cpu().numpy(), want[2])
    rel = (2 * ref.spread(l64, kw.get("scoring", "softmax")) + 16) * ref.F32
    nan = np.isnan(want[1])
    assert np.array_equal(nan, np.isnan(v))
    assert (np.abs(v - want[1]) <= rel * np.abs(want[1]) + 1e-45)[~nan].all(), np.abs(v - want[1]).max()
    return idx, w


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("T,E,k", [
    (1, 1, 1), (3, 2, 2), (1, 8, 2), (67, 7, 3), (130, 16, 4), (65, 33, 5), (300, 64, 8),
    (129, 65, 6), (77, 128, 16), (200, 160, 8), (131, 256, 8), (19, 257, 9), (33, 512, 10),
    (9, 1000, 70), (5, 1024, 1024), (2, 100, 100),
])
def test_choice_and_weights(scoring, dtype, T, E, k):
    l = logits_of(T, E, T + E, dtype)
    check(l, k, scoring=scoring)
    g = np.random.default_rng(7)
    bias = torch.from_numpy((0.1 * g.standard_normal(E)).astype(np.float32))
    check(l, k, scoring=scoring, bias=bias, scale=2.5)
    check(l, k, scoring=scoring, bias=torch.zeros(E), renormalize=False)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("group_top", [1, 2])
@pytest.mark.parametrize("T,E,G,tg,k", [
    (100, 256, 8, 4, 8), (33, 64, 8, 3, 6), (50, 160, 8, 3, 6), (41, 12, 6, 2, 4), (30, 96, 6, 4, 8),
    (64, 64, 64, 8, 8), (21, 512, 16, 4, 10), (9, 1020, 60, 7, 32), (10, 8, 2, 1, 4), (17, 192, 3, 1, 64),
    (7, 1024, 2, 1, 20), (40, 10, 5, 5, 10),
])
def test_groups(scoring, group_top, T, E, G, tg, k):
    for dtype in ("f32", "bf16"):
        l = logits_of(T, E, E + G, dtype)
        g = np.random.default_rng(9)
        bias = torch.from_numpy((0.1 * g.standard_normal(E)).astype(np.float32))
        check(l, k, scoring=scoring, groups=G, top_groups=tg, group_top=group_top, bias=bias)
        check(l, k, scoring=scoring, groups=G, top_groups=tg, group_top=group_top)


@pytest.mark.parametrize("E,G", [(8, 1), (64, 1), (64, 4), (256, 1), (256, 8), (100, 1)])
def test_ties_go_to_the_lowest_index(E, G):
    l = torch.zeros(40, E)
    l[1::3] = (torch.arange(E) % 3).float()
    l[2::3, E // 2:] = 1.0
    for bias in (None, torch.zeros(E), torch.full((E,), 0.25)):
        for scoring in ("softmax", "sigmoid"):
            check(l, 5, scoring=scoring, bias=bias, groups=G, top_groups=max(1, G // 2))


def test_near_ties_are_decided_in_64_bits():
    # keys that differ by a few 1e-9 around the border, next to each other in either order
    T, E, k = 64, 64, 8
    g = np.random.default_rng(11)
    base = g.standard_normal((T, 1)) * 0.1
    l = torch.from_numpy((base + g.permuted(np.tile(np.arange(E) * 4e-8, (T, 1)), axis=1)).astype(np.float32))
    bias = torch.from_numpy((1e-9 * g.standard_normal(E)).astype(np.float32))
    for scoring in ("softmax", "sigmoid"):
        for G in (1, 8):
            check(l, k, scoring=scoring, bias=bias, groups=G, top_groups=4 if G > 1 else 1)


def test_signed_zeros_tie():
    for dtype in ("f32", "bf16", "f16"):
        l = torch.zeros(30, 40, dtype=ref.TORCH[dtype])
        l[torch.from_numpy(np.random.default_rng(12).random((30, 40)) < 0.5)] = -0.0
        for bias in (None, torch.zeros(40), -torch.zeros(40)):
            for k in (3, 20):
                idx, _ = check(l, k, bias=bias)
                assert (idx.cpu() == torch.arange(k)).all()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_large_biases_near_ties(scoring):
    # f32 sums of score and bias have lost what decides: keys around +-1000, groups whose
    # two best cancel, and differences in the scores alone
    T, E, G = 64, 64, 8
    g = np.random.default_rng(19)
    l = torch.from_numpy((0.001 * g.standard_normal((T, E))).astype(np.float32))
    bias = torch.full((E,), -1000.0)
    bias[::8] = 1000.0
    check(l, 6, scoring=scoring, bias=bias, groups=G, top_groups=3)
    check(l, 12, scoring=scoring, bias=bias)
    check(l, 30, scoring=scoring, bias=torch.full((E,), 4096.0))


def test_scores_that_saturate():
    # equal in f32 (0 or 1), not in 64 bits
    l = torch.linspace(18, 30, 48).repeat(20, 1)
    l = l.gather(1, torch.from_numpy(np.random.default_rng(20).permuted(np.tile(np.arange(48), (20, 1)), axis=1)))
    for bias in (torch.zeros(48), torch.full((48,), 0.25)):
        check(l, 7, scoring="sigmoid", bias=bias, groups=4, top_groups=2)
        check(-l, 7, scoring="sigmoid", bias=torch.zeros(48))
        check(l * 8 - 200, 7, scoring="softmax", bias=torch.zeros(48))


@pytest.mark.parametrize("E,G", [(8, 1), (40, 4), (64, 8), (256, 8), (300, 1)])
def test_masked_experts_and_rows(E, G):
    for dtype in ("f32", "f16"):
        l = logits_of(90, E, 13, dtype)
        g = np.random.default_rng(14)
        l[torch.from_numpy(g.random((90, E)) < 0.6)] = -float("inf")
        l[3] = -float("inf")                      # nothing is left
        l[4] = -float("inf")
        l[4, E - 1] = 0.5                         # one expert is left
        l[5] = torch.finfo(l.dtype).min           # the lowest value is no mask
        l[6, 1:] = torch.finfo(l.dtype).min
        b = torch.from_numpy((0.2 * g.standard_normal(E)).astype(np.float32))
        for scoring in ("softmax", "sigmoid"):
            for bias in (None, b):
                idx, w = check(l, 4, scoring=scoring, bias=bias, groups=G, top_groups=max(1, G // 2))
                assert (idx[3] == -1).all() and (w[3] == 0).all()
                assert idx[4].tolist() == [E - 1, -1, -1, -1]


def test_nan_and_infinite_logits_show():
    l = logits_of(8, 32, 15, "f32")
    l[2, 9] = float("nan")
    l[5, 30] = float("inf")
    for scoring in ("softmax", "sigmoid"):
        for G in (1, 4):
            idx, w, _ = nm.route(l.cuda(), 4, scoring=scoring, groups=G, top_groups=1)
            assert ((idx >= 0) & (idx < 32)).all()
            assert torch.isnan(w[2]).all()
            ok = [0, 1, 3, 4, 6, 7]
            assert torch.isfinite(w[ok]).all()
            if scoring == "sigmoid":
                assert 9 in idx[2].tolist() and 30 in idx[5].tolist() and torch.isfinite(w[5]).all()


def test_far_logits():
    l = logits_of(50, 64, 16, "f32", std=30.0)
    check(l, 6, scoring="softmax")
    check(l, 6, scoring="sigmoid")
    check(l.half(), 6, scoring="softmax", renormalize=False)


def test_leading_dims_strides_and_empty():
    l = logits_of(24, 48, 17, "f32")
    check(l.view(2, 3, 4, 48), 4)
    wide = torch.zeros(24, 96)
    wide[:, ::2] = l
    check(wide[:, ::2], 4)
    i0, w0, c0 = nm.route(torch.empty(0, 16, device="cuda"), 4)
    assert i0.shape == (0, 4) and w0.shape == (0, 4) and c0.tolist() == [0] * 16
    i1, _, c1 = nm.route(l.cuda(), 4, counts=False)
    assert c1 is None and i1.shape == (24, 4)
    # logits that start at no multiple of 16 bytes
    for dtype in ("f32", "bf16"):
        flat = torch.empty(24 * 48 + 3, dtype=ref.TORCH[dtype], device="cuda")
        odd = flat[3:].view(24, 48)
        odd.copy_(l.to(ref.TORCH[dtype]))
        got = nm.route(odd, 4)
        want = nm.route(odd.clone(), 4)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_many_rows_count():
    # every block's histogram; rows past a multiple of every block size
    l = logits_of(20011, 24, 18, "bf16")
    idx, w, counts = nm.route(l.cuda(), 3, scoring="sigmoid", bias=torch.linspace(0, 0.3, 24).cuda())
    assert torch.equal(counts.cpu(), torch.bincount(idx.flatten().cpu(), minlength=24).int())
    again = nm.route(l.cuda(), 3, scoring="sigmoid", bias=torch.linspace(0, 0.3, 24).cuda())
    assert torch.equal(idx, again[0]) and torch.equal(w, again[1]) and torch.equal(counts, again[2])


# ---- the gradient ----------------------------------------------------------------

def check_grad(l, idx, dw, dtype, **kw):
    got = nm.route_backward(l.cuda(), idx.cuda(), dw.cuda(), **kw)
    torch.cuda.synchronize()
    assert got.shape == l.shape and got.dtype == l.dtype
    E, k = l.shape[-1], idx.shape[-1]
    l64 = l.double().numpy().reshape(-1, E)
    want, mag = ref.route_grad(l64, idx.numpy().reshape(-1, k), dw.double().numpy().reshape(-1, k), **kw)
    g = got.double().cpu().numpy().reshape(-1, E)
    # scores, their sums and products, as the weights' roundings twice over
    e = (4 * ref.spread(l64, kw.get("scoring", "softmax")) + 48) * ref.F32 * mag
    tol = e + ref.HALF[dtype] * (np.abs(want) + e) + max(ref.TINY[dtype], 1e-45)
    over = np.abs(g - want) > tol
    assert not over.any(), (np.argwhere(over)[0], g[over][0], want[over][0])
    return got


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("dtype,T,E,k", [
    ("f32", 1, 1, 1), ("f32", 5, 8, 2), ("bf16", 67, 16, 4), ("f16", 33, 33, 5), ("f32", 100, 64, 8),
    ("bf16", 41, 160, 6), ("f32", 70, 256, 8), ("f16", 9, 300, 12), ("f32", 3, 1024, 40), ("f32", 2, 100, 100),
])
def test_gradient(scoring, renormalize, dtype, T, E, k):
    l = logits_of(T, E, 20 + E, dtype)
    l[T // 2, : E // 2] = -float("inf")
    idx, _, _ = nm.route(l.cuda(), k, scoring=scoring)
    dw = torch.from_numpy(np.random.default_rng(21).standard_normal((T, k)).astype(np.float32))
    check_grad(l, idx.cpu(), dw, dtype, scoring=scoring, renormalize=renormalize, scale=1.5)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_gradient_empty_rows_and_foreign_slots(scoring):
    l = logits_of(20, 24, 22, "f32")
    l[7] = -float("inf")
    idx = torch.from_numpy(np.random.default_rng(23).integers(0, 24, (20, 3)).astype(np.int32))
    idx[:, 1] = (idx[:, 0] + 5) % 24
    idx[:, 2] = (idx[:, 0] + 11) % 24
    idx[3] = -1                              # an empty row
    idx[4, 0] = -1
    idx[5, 1] = 24                           # no expert
    idx[6] = torch.tensor([2 ** 31 - 1, -2 ** 31, 3], dtype=torch.int32)
    idx[8] = torch.tensor([4, 4, 9], dtype=torch.int32)  # named twice: both count
    dw = torch.randn(20, 3, generator=torch.Generator().manual_seed(1))
    got = check_grad(l, idx, dw, "f32", scoring=scoring)
    assert (got[3] == 0).all() and (got[7] == 0).all()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_gradient_against_differences(scoring, renormalize):
    # the weights' change along a direction, from the definition in 64 bits
    T, E, k = 12, 20, 4
    l = logits_of(T, E, 25, "f32")
    kw = dict(scoring=scoring, renormalize=renormalize, scale=1.7)
    idx, _, _ = nm.route(l.cuda(), k, **kw)
    g = np.random.default_rng(26)
    dw, u = g.standard_normal((T, k)).astype(np.float32), g.standard_normal((T, E))
    got = nm.route_backward(l.cuda(), idx, torch.from_numpy(dw).cuda(), **kw).double().cpu().numpy()
    l64, i = l.double().numpy(), idx.cpu().numpy()

    def weights(at):
        s = np.stack([ref.scores(r, scoring) for r in at])
        v = np.take_along_axis(s, i, 1)
        return 1.7 * (v / (v.sum(1, keepdims=True) + 1e-9) if renormalize else v)

    step = 1e-5
    diff = ((weights(l64 + step * u) - weights(l64 - step * u)) / (2 * step) * dw).sum()
    # the differences are exact to step^2; the gradient's f32 errors are 1e-6 of its terms
    assert abs((got * u).sum() - diff) <= 1e-8 + 4e-6 * np.abs(got * u).sum()


def test_in_place_gradient_graph_and_streams():
    T, E, k = 700, 96, 6
    l = logits_of(T, E, 27, "bf16").cuda()
    bias = torch.linspace(-0.1, 0.1, E, device="cuda")
    dw = torch.randn(T, k, device="cuda")

    def both():
        idx, w, c = nm.route(l, k, scoring="sigmoid", bias=bias, groups=4, top_groups=2)
        return idx, w, c, nm.route_backward(l, idx, dw, scoring="sigmoid")

    want = [t.clone() for t in both()]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        both()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=s):
            got = both()
    keep = l.clone()
    for n in range(4):
        l.copy_(keep.flip(0) if n % 2 else keep)
        for t in got:
            t.fill_(7)
        graph.replay()
        eager = both()   # between the replays, on the default stream after it
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager))
        if n % 2 == 0:
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    # dlogits in the logits' own buffer, through the C call
    idx = want[0]
    rc = nm._lib.lib().nomas_route_backward(1, l.data_ptr(), idx.data_ptr(), dw.data_ptr(), T, E, k, 1, 1, 1.0,
                                            1e-9, l.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    l2 = keep.flip(0)  # (the last replay's)
    assert torch.equal(l, nm.route_backward(l2, idx, dw, scoring="sigmoid"))


def test_two_streams_at_once():
    l = [logits_of(4000, 128, 30 + i, "f32").cuda() for i in range(2)]
    b = torch.linspace(-0.1, 0.1, 128, device="cuda")
    want = [nm.route(x, 6, scoring="sigmoid", bias=b) for x in l]
    torch.cuda.synchronize()
    s = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = []
        for x, st in zip(l, s):
            with torch.cuda.stream(st):
                got.append(nm.route(x, 6, scoring="sigmoid", bias=b))
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for u, v in zip(got, want) for p, q in zip(u, v))


def test_gradient_of_repeated_experts_has_the_same_bits():
    l = logits_of(64, 32, 33, "f32").cuda()
    idx = torch.from_numpy(np.random.default_rng(34).integers(0, 4, (64, 16)).astype(np.int32)).cuda()
    dw = torch.randn(64, 16, device="cuda", generator=torch.Generator("cuda").manual_seed(3))
    for scoring in ("softmax", "sigmoid"):
        want = nm.route_backward(l, idx, dw, scoring=scoring)
        check_grad(l.cpu(), idx.cpu(), dw.cpu(), "f32", scoring=scoring)
        assert all(torch.equal(nm.route_backward(l, idx, dw, scoring=scoring), want) for _ in range(3))


def plain_choice(l, k, scoring, bias, groups, top_groups, group_top):
    """The choice in f64 torch operations, for many rows at once."""
    T, E = l.shape
    s = torch.sigmoid(l.double()) if scoring == "sigmoid" else torch.softmax(l.double(), -1)
    key = l.double() if bias is None and groups == 1 else s if bias is None else s + bias.double()
    out = l == -float("inf")
    key = key.masked_fill(out, -float("inf"))
    if groups > 1:
        best = key.view(T, groups, -1).sort(-1, descending=True).values[..., :group_top]
        score = best.masked_fill(best == -float("inf"), 0).sum(-1)
        score = score.masked_fill(best[..., 0] == -float("inf"), -float("inf"))
        kept = score.sort(dim=-1, descending=True, stable=True).indices[:, :top_groups]
        keep = torch.zeros(T, groups, dtype=torch.bool, device=l.device).scatter_(1, kept, True)
        key = key.masked_fill(~keep.repeat_interleave(E // groups, 1), -float("inf"))
    top = key.sort(dim=-1, descending=True, stable=True)
    idx = top.indices[:, :k].masked_fill(top.values[:, :k] == -float("inf"), E).sort(-1).values
    return idx.masked_fill(idx == E, -1).int()


@pytest.mark.parametrize("seed", range(40))
def test_crowded_borders(seed):
    # logits and biases of few levels, a few of them moved by an f32 step or so: ties and
    # near ties at the borders of experts and groups in most rows
    g = np.random.default_rng(1000 + seed)
    G = int(g.choice([1, 1, 2, 4, 5, 8, 16]))
    E = G * int(g.integers(2, max(3, min(600, 1024) // G)))
    tg = int(g.integers(1, G + 1))
    k = int(min(g.choice([1, 2, 4, 8, 8, 12, 16, 17, 40]), E // G * tg))
    T = int(g.choice([7, 300, 3000]))
    levels = int(g.choice([2, 5, 40, 400]))
    l = torch.from_numpy((g.integers(-levels, levels + 1, (T, E)) * (3.0 / levels)).astype(np.float32))
    moved = torch.from_numpy(g.random((T, E)) < 0.2)
    l = torch.where(moved, l * (1 + 2.0 ** -22 * torch.from_numpy(g.integers(-2, 3, (T, E)).astype(np.float32))), l)
    l[torch.from_numpy(g.random((T, E)) < 0.05)] = -float("inf")
    l = l.to(ref.TORCH[str(g.choice(["f32", "f32", "bf16", "f16"]))]).cuda()
    bias = [None, torch.zeros(E), torch.from_numpy((g.integers(-3, 4, E) * 0.05).astype(np.float32)),
            torch.from_numpy((100 * g.standard_normal(E)).astype(np.float32))][int(g.integers(4))]
    bias = None if bias is None else bias.cuda()
    for scoring in ("sigmoid", "softmax"):
        for top in (1, 2):
            idx, w, counts = nm.route(l, k, scoring=scoring, bias=bias, groups=G, top_groups=tg, group_top=top)
            want = plain_choice(l, k, scoring, bias, G, tg, top)
            bad = (idx != want).any(1).nonzero().flatten()
            assert not bad.numel(), (E, G, tg, k, levels, scoring, top, int(bad[0]), idx[bad[0]], want[bad[0]])
            assert torch.equal(counts, torch.bincount(want[want >= 0], minlength=E).int())
