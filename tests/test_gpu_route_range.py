"""Routing and its gradient on the GPU where f32 has little left: gradients in which all
but eps' share cancels, scores that underflow, empty slots' values.

Against the definitions in 80-bit long doubles, whose range holds every score here
and whose digits outlast the cancellation."""
import numpy as np
import pytest
import torch

import nomas_moe as nm
import _block_ops as ref
from test_gpu_route import logits_of

pytestmark = pytest.mark.gpu


def values(T, k, seed):
    return torch.from_numpy(np.random.default_rng(seed).standard_normal((T, k)).astype(np.float32))


@pytest.mark.parametrize("dw", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("k", [2, 12])
def test_an_empty_slots_value_is_not_read(scoring, k, dw):
    # as the routed experts do with its weight
    l = logits_of(9, 40, 3, "f32")
    l[8, 3] = -float("inf")
    idx = torch.arange(k, dtype=torch.int32).repeat(9, 1) * 3
    d = values(9, k, 4)
    for r, none in enumerate((-1, 40, 2 ** 31 - 1, -2 ** 31)):
        idx[2 * r, r % k] = none
        d[2 * r, r % k] = dw
    idx[1], d[1] = -1, dw                      # nothing but empty slots
    d[8, 1] = dw                               # a masked expert's slot is an empty one
    idx[8, 1] = 3
    for renormalize in (True, False):
        got = nm.route_backward(l.cuda(), idx.cuda(), d.cuda(), scoring=scoring, renormalize=renormalize)
        clean = torch.where(torch.isfinite(d), d, 0.0)
        want = nm.route_backward(l.cuda(), idx.cuda(), clean.cuda(), scoring=scoring, renormalize=renormalize)
        assert torch.isfinite(got).all() and torch.equal(got, want)
        assert (got[1] == 0).all() and got[8, 3] == 0


# ---- weights of scores that underflow -----------------------------------------------

X = np.longdouble


def scores(row, scoring):
    row = row.astype(X)
    if scoring == "sigmoid":
        return 1 / (1 + np.exp(-row))
    e = np.exp(row - row.max()) if np.isfinite(row.max()) else np.zeros_like(row)
    return e / e.sum() if e.any() else e


def weights(logits, idx, scoring, scale, eps):
    w = np.zeros(idx.shape, X)
    for r in range(logits.shape[0]):
        s = scores(logits[r], scoring)
        sel = idx[r] >= 0
        v = s[idx[r][sel]]
        w[r, sel] = scale * v / (v.sum() + X(eps))
    return w


def check_weights(l, k, scoring, eps, scale=2.5, **kw):
    """An exponential's error is its argument's in half steps, for the score, the sum and eps' share
    in it, and the products and sums (trees) come to 64 more."""
    idx, w, _ = nm.route(l.cuda(), k, scoring=scoring, eps=eps, scale=scale, **kw)
    i, w = idx.cpu().numpy(), w.double().cpu().numpy()
    l64 = l.double().numpy()
    want = weights(l64, i, scoring, scale, np.float32(eps))
    rel = (4 * ref.spread(l64, scoring) + 64) * ref.F32
    over = ~(np.abs(w - want) <= rel * want + 2.0 ** -147)
    assert not over.any(), (over.sum(), np.argwhere(over)[0], w[over][0], float(want[over][0]))
    return i


@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-9, 1e-2])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("E,k", [(16, 1), (16, 4), (64, 8), (40, 20), (256, 30)])
def test_weights_of_chosen_scores_that_underflow(eps, dtype, E, k):
    l = logits_of(30, E, E + k, dtype, std=3.0)
    # a sigmoid of nothing but low logits
    for low in (20.0, 95.0, 130.0, 300.0):
        check_weights((l.double() - low).to(l.dtype), k, "sigmoid", eps)
    # a softmax whose bias chooses experts far below the best ones; likewise groups
    bias = torch.zeros(E)
    bias[E // 2:] = 10.0
    for low in (20.0, 95.0, 130.0, 300.0, 1000.0):
        far = l.double()
        far[:, E // 2:] -= low
        far = far.to(l.dtype)
        i = check_weights(far, min(k, E // 2), "softmax", eps, bias=bias.cuda())
        assert (i >= E // 2).all()
        check_weights(far, min(k, E // 2), "softmax", eps, bias=bias.cuda(), groups=2, top_groups=1)


def test_weights_of_masked_rows_without_eps():
    l = logits_of(6, 24, 5, "f32")
    l[1] = -float("inf")
    l[2, 1:] = -float("inf")
    l[3, 2:] = -float("inf")
    l[3, :2] = -200.0
    for scoring in ("softmax", "sigmoid"):
        check_weights(l, 4, scoring, 0.0)


# ---- gradients in which all but eps' share cancels -----------------------------------

def grad(logits, idx, dw, scoring, renormalize, scale, eps):
    """(dlogits, magnitudes, own): the definition, and the size of the terms that it has when it is
    written without cancellation.  A chosen expert i has scale s_i / S^2 times
    sum_j s_j (d_i - d_j) + eps d_i (a softmax: times the scores not chosen): its terms' magnitudes.
    own: the roundings of this very evaluation, 2^-64 of the terms that cancel in it, for each of the E + k
    terms of its sums and 8 operations besides (all there is where eps is 0: without a second slot the
    gradient is 0 then)."""
    T, E = logits.shape
    dl, mag, own = np.zeros((T, E), X), np.zeros((T, E), X), np.zeros((T, E), X)
    for r in range(T):
        s = scores(logits[r], scoring)
        sel = [(e, X(dw[r, t])) for t, e in enumerate(idx[r]) if 0 <= e < E and logits[r, e] != -np.inf]
        if not sel:
            continue
        S = sum(s[e] for e, _ in sel) + X(eps) if renormalize else X(1)
        A = sum(s[e] * d for e, d in sel)
        B = sum(s[e] * abs(d) for e, d in sel)
        ds = np.zeros(E, X)
        for e, d in sel:
            ds[e] += scale * ((d - A / S) / S if renormalize else d)
        chosen = {e for e, _ in sel}
        rest = sum(s[e] for e in range(E) if e not in chosen)
        if scoring == "sigmoid":
            dl[r] = ds * s * (1 - s)
        else:
            dl[r] = s * (ds - (s * ds).sum())
            mag[r] = s * scale * B * (X(eps) / S / S if renormalize else 1)
        for e, d in sel:
            others = sum(s[f] * abs(d - g) for f, g in sel)
            if renormalize:
                left = X(eps) * abs(d) * (rest if scoring == "softmax" else 1)
                m = (others * (1 + X(eps)) + left) / S / S
            else:
                m = others + rest * abs(d) if scoring == "softmax" else abs(d)
            slope = scale * s[e] * ((1 - s[e]) if scoring == "sigmoid" else 1)
            mag[r, e] = slope * m
            noise = X(2) ** -64 * (E + len(sel) + 8) * scale * 2 * (abs(d) + B / S) / S  # of ds[e]
            own[r, e] += s[e] * noise
            if scoring == "softmax":
                own[r] += s * s[e] * noise     # by way of the inner product
    return dl, mag, own


def check_grad(l, idx, dw, dtype="f32", scoring="softmax", renormalize=True, scale=1.5, eps=1e-9):
    """The kernel sums differences from the dominant slot's value; against the terms above,
    differences from each slot's own, their magnitudes are 3 k + 5 times as large at most
    (|d_i - c| <= (k + 1) of them, since the dominant score is a (k + 1)-th of the sum; the sum
    of the others' and eps' share as much again).  Their roundings: exponentials, whose arguments'
    errors are `spread` half steps, sums (trees) and quotients, 48 besides."""
    got = nm.route_backward(l.cuda(), idx.cuda(), dw.cuda(), scoring=scoring, renormalize=renormalize, scale=scale,
                            eps=eps).double().cpu().numpy()
    k = idx.shape[1]
    l64 = l.double().numpy()
    want, mag, own = grad(l64, idx.numpy(), dw.double().numpy(), scoring, renormalize, scale, np.float32(eps))
    e = (4 * ref.spread(l64, scoring) + 48) * ref.F32 * (3 * k + 5) * mag
    tol = e + ref.HALF[dtype] * (np.abs(want) + e) + max(ref.TINY[dtype], 2.0 ** -148) + own
    over = ~(np.abs(got - want) <= tol)
    assert not over.any(), (over.sum(), np.argwhere(over)[0], got[over][0], float(want[over][0]), float(tol[over][0]))
    return got


def route_of(l, k, scoring):
    return nm.route(l.cuda(), k, scoring=scoring, counts=False)[0].cpu()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("eps", [1e-9, 1e-2, 1.0])
@pytest.mark.parametrize("dtype,E", [("f32", 2), ("f32", 16), ("bf16", 64), ("f16", 100), ("f32", 256), ("f32", 1000)])
def test_gradient_of_a_single_survivor(scoring, eps, dtype, E):
    l = logits_of(33, E, E, dtype)
    got = check_grad(l, route_of(l, 1, scoring), values(33, 1, E), dtype, scoring, eps=eps)
    if dtype == "f32":
        assert (got != 0).any(1).all()
    # the same with slots to spare, all but one expert masked
    k = min(E, 6)
    for r in range(33):
        keep = l[r, r % E].clone()
        l[r] = -float("inf")
        l[r, r % E] = keep
    idx = route_of(l, k, scoring)
    assert ((idx >= 0).sum(1) == 1).all()
    check_grad(l, idx, values(33, k, E + 1), dtype, scoring, eps=eps)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("eps", [1e-9, 1e-2])
@pytest.mark.parametrize("E,k", [(8, 2), (64, 8), (100, 20), (256, 8), (1024, 70)])
def test_gradient_of_equal_values_and_dominant_experts(scoring, eps, E, k):
    T = 21
    l = logits_of(T, E, E + k, "f32")
    l[::3, E // 3] = 9.0                       # nearly all of the row's weight
    l[1::3] -= 12.0                            # (sigmoid: eps beside small scores)
    idx = route_of(l, k, scoring)
    d = values(T, k, E)
    check_grad(l, idx, d, "f32", scoring, eps=eps)
    d[:, :] = d[:, :1]                         # no weight can gain from another
    check_grad(l, idx, d, "f32", scoring, eps=eps)
    d[:, k // 2] += 1e-3
    check_grad(l, idx, 1000 + d, "f32", scoring, eps=eps)
    check_grad(l, idx, d, "f32", scoring, renormalize=False)


@pytest.mark.parametrize("dtype,E,k", [("f32", 16, 4), ("bf16", 64, 8), ("f32", 256, 40)])
def test_gradient_of_scores_that_are_not_renormalised(dtype, E, k):
    # all of the softmax's weight on the chosen: what is left is the rest's share
    l = logits_of(18, E, 7, dtype)
    l[:, :k] += 10.0
    idx = route_of(l, k, "softmax")
    d = values(18, k, 8)
    check_grad(l, idx, d, dtype, "softmax", renormalize=False)
    check_grad(l, idx, d[:, :1].repeat(1, k), dtype, "softmax", renormalize=False)


def test_gradient_of_a_training_step_keeps_its_digits():
    # top-1 of a batch: the 2-norm's error, not only each element's bound
    l = logits_of(4000, 64, 9, "f32")
    for scoring in ("softmax", "sigmoid"):
        idx, d = route_of(l, 1, scoring), values(4000, 1, 10)
        got = nm.route_backward(l.cuda(), idx.cuda(), d.cuda(), scoring=scoring).double().cpu().numpy()
        want, _, _ = grad(l.double().numpy(), idx.numpy(), d.double().numpy(), scoring, True, 1.0, np.float32(1e-9))
        assert np.linalg.norm((got - want).astype(float)) <= 1e-5 * np.linalg.norm(want.astype(float))


# ---- gradients of scores that underflow ------------------------------------------------

@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-9])
@pytest.mark.parametrize("E,k", [(16, 1), (16, 4), (64, 8), (256, 30)])
def test_gradient_of_scores_that_underflow(scoring, eps, E, k):
    l = logits_of(20, E, E + k, "f32", std=2.0)
    idx = torch.from_numpy(np.random.default_rng(k).permuted(np.tile(np.arange(E // 2, dtype=np.int32), (20, 1)), axis=1)
                           [:, :k] + E // 2)
    for low in (20.0, 95.0, 130.0, 300.0):
        far = l.clone()
        if scoring == "sigmoid":
            far -= low
        else:
            far[:, E // 2:] -= low             # chosen far below the row's best
        check_grad(far, idx, values(20, k, 11), "f32", scoring, eps=eps)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_gradient_of_masked_choices_without_eps(scoring):
    l = logits_of(5, 24, 12, "f32")
    l[1] = -float("inf")
    l[2, 3] = l[2, 5] = -float("inf")
    idx = torch.tensor([[1, 2], [3, 5], [3, 5], [-1, -1], [3, 4]], dtype=torch.int32)
    got = check_grad(l, idx, values(5, 2, 13), "f32", scoring, eps=0.0)
    assert (got[1:4] == 0).all()


# ---- groups ------------------------------------------------------------------------

@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_group_scores_past_f32(scoring, sign):
    # sums of two biases near the largest f32: infinite in 32 bits, told apart in 64
    l = logits_of(9, 32, 14, "f32")
    bias = torch.zeros(32)
    for g, top in enumerate((3.0e38, 3.2e38, 2.9e38, 3.1e38)):
        bias[8 * g:8 * g + 8] = sign * top
    idx, _, _ = nm.route(l.cuda(), 4, scoring=scoring, bias=bias.cuda(), groups=4, top_groups=1)
    best = 1 if sign > 0 else 2
    assert (idx // 8 == best).all()
