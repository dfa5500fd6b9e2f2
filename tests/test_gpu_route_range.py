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
