"""forward_few on 8-bit weights with activations near the ends of bf16's range.

The gates are 1 (weights 0, biases 1), so that the hidden activations are as large as the up products and
the bounds of test_gpu_few hold as they are.
"""
import numpy as np
import pytest
import torch

import nomas_moe as nm
import _fp8 as F
from _common import rounded, small_case
from _gpu import layer_from_tensors, to_device
from test_gpu_few import near, plain

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fp8", [True, False])
# x, up and down weights are 2^each times numbers near 1
@pytest.mark.parametrize("ex,eu,ed", [(121, -20, 0), (121, 0, -10), (-115, 0, 0), (4, 115, -115)])
@pytest.mark.parametrize("rows,D,E,k,H,s", [(1, 256, 4, 2, 264, 0.0), (20, 264, 4, 2, 128, 0.5), (64, 256, 4, 1, 300, 0.0),
                                            (64, 512, 2, 2, 512, 0.0)])
def test_range(rows, D, E, k, H, s, ex, eu, ed, fp8):
    t, x = small_case(rows, D, E, k, H, rows + D, dense=s > 0, router_std=0.1)
    for n in t:
        if "gate" in n:
            t[n] = np.full_like(t[n], 1.0 if "bias" in n else 0.0)
        elif "up" in n or "down" in n:
            t[n] = np.zeros_like(t[n]) if "bias" in n else np.ldexp(t[n], eu if "up" in n else ed)
    x = x.copy()
    x[::2] = np.ldexp(x[::2], ex)  # the other rows as they are
    layer = layer_from_tensors(t, "bf16", D, H, E, k, s)
    rt, xm = rounded(t, x, "bf16")
    p, dense = nm.workloads.oracle_params(rt, E)
    names = ("wg", "bg", "wu", "bu", "wd", "bd")
    ffn = [[np.asarray(p[n][e], np.float64) for n in names] for e in range(E)]
    ffn += [[np.asarray(dense[n], np.float64) for n in names]] if s > 0 else []
    if fp8:
        layer.quantize()
        for f in ffn:
            for i in (0, 2, 4):
                q, c = F.quantize(torch.from_numpy(f[i]), True)
                f[i] = (q * F.expand(c, *q.shape, True)).numpy()
    r = np.random.default_rng(rows)
    idx = np.stack([r.permutation(E)[:k] for _ in range(rows)]).astype(np.int32)
    w = r.random((rows, k)).astype(np.float32)
    y = layer.forward_few(to_device(x, "bf16"), torch.from_numpy(idx).cuda(), torch.from_numpy(w).cuda(), fp8=fp8)
    want, off = plain(xm, ffn, idx, w, "bf16", s)
    assert np.abs(want).max() < 2.0 ** 127
    near(y, want, off)
