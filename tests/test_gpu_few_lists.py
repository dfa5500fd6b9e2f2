"""forward_few under the caller's routing where a call has more slots than the lists keep in LDS (2,048).

The bound is test_gpu_few's with the sum of an expert's weights counted: up to top_k numbers added in f32
are off by at most top_k steps of 2^-24 of their magnitudes' sum, times the expert's output.
"""
import numpy as np
import pytest
import torch

from test_gpu_few import HALF, case, near, plain

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,fp8", [("f32", False), ("bf16", False), ("f16", True)])
@pytest.mark.parametrize("rows,D,E,k,H,s", [(64, 40, 64, 64, 24, 0.0), (64, 72, 256, 40, 40, 0.5), (33, 64, 100, 70, 16, 0.0),
                                            (64, 64, 32, 32, 24, 0.25)])
def test_many_slots(rows, D, E, k, H, s, dtype, fp8):
    layer, x, xm, ffn = case(rows, D, E, k, H, dtype, 500 + rows + D, s, fp8)
    r = np.random.default_rng(rows + E)
    idx = r.integers(-2, E + 1, (rows, k)).astype(np.int32)  # empty slots, repeated experts, any order
    idx[1], idx[2, ::2] = 3, 5  # one expert in every slot, one in every other
    idx[rows // 2] = -1  # a row with nothing
    w = r.normal(size=(rows, k)).astype(np.float32)
    w[idx < 0] = np.nan  # what stands beside an empty slot is not used
    w[idx >= E] = np.inf
    live = (idx >= 0) & (idx < E)
    used, named = np.where(live, w, 0), np.where(live, idx, -1)
    y = layer.forward_few(x, torch.from_numpy(idx).cuda(), torch.from_numpy(w).cuda(), fp8=fp8)
    want, off = plain(xm, ffn, named, used, dtype, s)
    x64 = xm.astype(np.float64)
    for e, (wg, bg, wu, bu, wd, bd) in enumerate(ffn[:E]):
        g = x64 @ wg.T + bg
        out = (g / (1 + np.exp(-g)) * (x64 @ wu.T + bu)) @ wd.T + bd
        size = np.where(named == e, np.abs(used), 0).sum(1)
        off += (1 + HALF[dtype]) * k * 2.0 ** -24 * size[:, None] * np.abs(out)
    near(y, want, off)
    if s == 0.0:
        assert not y[rows // 2].any()
    # the first 2,048 slots or fewer alone: the same lists from LDS
    n = 2048 // k
    part = layer.forward_few(x[:n], torch.from_numpy(idx[:n]).cuda(), torch.from_numpy(w[:n]).cuda(), fp8=fp8)
    near(part, want[:n], off[:n])
