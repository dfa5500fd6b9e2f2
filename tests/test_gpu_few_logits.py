"""forward_few's choice on logits so large that f32 does not hold their differences, or the logits themselves.

A weight is an exponential of a difference of logits over a sum of them: the difference is exact here, and an
exponential (2 steps of 2^-23), its sum over 256 experts in a tree (10 roundings), a division and two
products round: 16 steps of 2^-23 at most.
"""
import numpy as np
import pytest
import torch

from _common import small_case
from _gpu import layer_from_tensors

pytestmark = pytest.mark.gpu


def check(layer, x, wr, k, E):
    layer.forward_few(x)
    idx, w, counts, _ = layer.routing(len(x))
    logits = x.double().cpu().numpy() @ wr.astype(np.float64).T
    for i in range(len(x)):
        order = sorted(range(E), key=lambda e: (-logits[i, e], e))
        assert list(idx[i]) == sorted(order[:k])
        p = np.exp(logits[i] - logits[i].max())
        want = p[idx[i]] / (p[idx[i]].sum() + 1e-9 * p.sum())
        assert np.allclose(w[i], want, rtol=16 * 2.0 ** -23, atol=2.0 ** -126)
    assert counts.sum() == len(x) * k


def layer_of(wr, E, k, dtype):
    t, _ = small_case(1, wr.shape[1], E, k, 16, 11)
    t["blocks.0.moe.router.weight"] = wr
    return layer_from_tensors(t, dtype, wr.shape[1], 16, E, k, 0.0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [2, 40])
@pytest.mark.parametrize("E,k", [(4, 2), (16, 3), (64, 8), (200, 6), (256, 40)])
def test_differences_that_f32_does_not_hold(rows, E, k, dtype):
    """Logits of +-(2^34 + 2^10) and a small part: f32's steps are 2^11 there."""
    r = np.random.default_rng(E + k)
    wr = np.zeros((E, 64), np.float32)
    # (the large column apart from the others by 32: 16-bit products are summed in f32 32 at a time)
    wr[:, 0], wr[:, 40], wr[:, 41] = 2.0 ** 17, 2.0 ** 5, r.permutation(E) / 4
    x = torch.zeros(rows, 64)
    x[:, 0], x[:, 40], x[:, 41] = 2.0 ** 17, 2.0 ** 5, 1.0
    x[1::2, 0] *= -1
    check(layer_of(wr, E, k, dtype), x.to(torch.bfloat16 if dtype == "bf16" else torch.float32).cuda(), wr, k, E)


@pytest.mark.parametrize("rows", [2, 40])
@pytest.mark.parametrize("E,k", [(4, 2), (16, 3), (64, 8), (200, 6)])
def test_logits_past_f32(rows, E, k):
    """Logits of 2^160 (every third expert's), -2^160 or 0."""
    wr = np.zeros((E, 64), np.float32)
    wr[:, 0] = np.where(np.arange(E) % 3 == 1, 2.0 ** 60, 0)
    x = torch.zeros(rows, 64)
    x[:, 0] = 2.0 ** 100
    x[1::2, 0] *= -1
    check(layer_of(wr, E, k, "f32"), x.cuda(), wr, k, E)
