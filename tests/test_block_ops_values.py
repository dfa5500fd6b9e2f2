"""Scalars of the routing and the block seams that f32 does not hold, and tensors that the
Python mirror has to refuse by its own error -- CPU only."""
import pytest
import torch

import nomas_moe as nm
from nomas_moe import _lib
from test_block_ops_refusals import BACK, P, SEAM, fake, lib, no_lib, refused, route  # noqa: F401


@pytest.mark.parametrize("kw,text", [
    (dict(scale=1e39), "scale"), (dict(scale=-1e300), "scale"), (dict(eps=1e39), "eps"), (dict(eps=1e300), "eps"),
])
def test_route_scalars_past_f32(kw, text):
    assert route(**kw) == 2
    assert text in _lib.last_error() and "f32" in _lib.last_error()
    a = dict(dtype=0, logits=P, idx=P, dw=P, rows=4, experts=8, k=2, scoring=0, renorm=1, scale=1.0, eps=1e-9, dl=P)
    assert lib().nomas_route_backward(*{**a, **kw}.values(), None) == 2
    assert text in _lib.last_error() and "f32" in _lib.last_error()


@pytest.mark.parametrize("kw,text", [
    (dict(alpha=1e39), "residual_scale"), (dict(alpha=-1e300), "residual_scale"), (dict(eps=1e-39), "eps"),
    (dict(eps=1e-50), "eps"),
])
def test_seam_scalars_that_f32_does_not_hold(kw, text):
    assert lib().nomas_block_seam(*{**SEAM, **kw}.values(), None) == 2
    assert text in _lib.last_error()
    assert lib().nomas_block_seam_backward(*{**BACK, **kw}.values(), None) == 2
    assert text in _lib.last_error()


def test_scalars_at_the_ends_of_f32_are_taken():
    none = dict(rows=0, logits=None, idx=None, w=None)
    assert route(**none, scale=3e38, eps=3e38) == 0 and route(**none, scale=-3e38, eps=0.0) == 0
    none = dict(rows=0, x=None, y=None, out=None, h=None)
    for eps in (0.0, 2.0 ** -126, 3e38):
        assert lib().nomas_block_seam(*{**SEAM, **none, "eps": eps, "alpha": 3e38}.values(), None) == 0


def test_the_mirrors_own_error_for_types_and_shapes(no_lib):  # noqa: F811
    x64 = fake(2, 3, 16, dtype=torch.float64)
    refused("f32, bf16 or f16", nm.block_seam, x64, x64)
    refused("f32, bf16 or f16", nm.block_seam_backward, x64, x64, x64, x64)
    refused("f32, bf16 or f16", nm.norm_modulate, x64, fake(2, 16), fake(2, 16))
    refused("f32, bf16 or f16", nm.gated_residual, x64, x64, fake(2, 16))
    # a row of logits with a choice that has no slots' dimension
    refused("idx", nm.route_backward, fake(8), fake(1, dtype=torch.int32)[0], fake(1)[0])
    refused("dw", nm.route_backward, fake(8), fake(2, dtype=torch.int32), fake(1)[0])


# 6 rows of 64 bf16 are 768 bytes, 4 rows of 8 f32 128: tensors that lie nearer share memory
APART = {**SEAM, "y": 2 * P, "out": 3 * P, "h": 4 * P}


@pytest.mark.parametrize("kw", [
    dict(out=P + 128), dict(out=P - 640), dict(out=2 * P + 16), dict(out=2 * P - 752), dict(h=P + 640),
    dict(h=2 * P - 128), dict(h=3 * P + 16), dict(out=4 * P + 752), dict(out=P, y=P + 256),
])
def test_seam_outputs_that_share_part_of_a_tensor(kw):
    assert lib().nomas_block_seam(*{**APART, **kw}.values(), None) == 2
    assert "overlap" in _lib.last_error()


@pytest.mark.parametrize("kw", [
    dict(dx=P + 128), dict(dx=2 * P + 256), dict(dy=P + 752), dict(dh=2 * P + 16), dict(y=3 * P, dy=3 * P - 512),
])
def test_seam_gradients_that_share_part_of_a_tensor(kw):
    assert lib().nomas_block_seam_backward(*{**BACK, **kw}.values(), None) == 2
    assert "overlap" in _lib.last_error()


@pytest.mark.parametrize("dl", [P + 4, P + 124, P - 32])
def test_route_gradient_that_shares_part_of_the_logits(dl):
    a = dict(dtype=0, logits=P, idx=P, dw=P, rows=4, experts=8, k=2, scoring=0, renorm=1, scale=1.0, eps=1e-9, dl=dl)
    assert lib().nomas_route_backward(*a.values(), None) == 2
    assert "overlap" in _lib.last_error()
