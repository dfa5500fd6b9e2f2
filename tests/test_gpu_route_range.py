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
