"""The block seam's gradients on rows of very large and very small values, whose
squares f32 still holds but not the powers that the formulas have of their norms."""
import pytest
import torch

import nomas_moe as nm
import _block_ops as ref
from test_gpu_block_seam import dev, inputs, wide, NAMES

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,S,D", [(1, 6, 96), (2, 30, 520), (40, 3, 1032)])
@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-6])
@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("size", [1e16, 1e15, 1e12, 1e-12, 1e-15])
def test_gradients_of_large_and_small_rows(dtype, B, S, D, eps, post, size):
    t = inputs(B, S, D, dtype, D + S, NAMES)
    t["out"], t["y"] = t["out"] * size, t["y"] * size
    pw = t["post_w"] if post else None
    got = nm.block_seam_backward(*(dev(t[n]) for n in (*NAMES, "gate", "scale")), post_norm=post, post_w=dev(pw),
                                 norm_w=dev(t["norm_w"]), residual_scale=0.5, eps=eps)
    want, mag = ref.seam_grad(*(wide(t[n]) for n in (*NAMES, "gate", "scale")), post, wide(pw), wide(t["norm_w"]), 0.5,
                              eps)
    for n, w in want.items():
        off = (got[n].double().cpu() - w).abs() - ref.seam_grad_bound(n, w, mag[n], B * S, dtype)
        assert (off <= 0).all(), (n, float(off.max()), float(w.abs().max()))
