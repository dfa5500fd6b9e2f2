"""What a forward_few call leaves behind for the next call on its layer."""
import pytest
import torch

import nomas_moe as nm
from nomas_moe import _lib
from test_gpu_few import case

pytestmark = pytest.mark.gpu

NOTHING = {
    "forward": lambda l, x, i, w: l.forward(x),
    "forward of a host tensor": lambda l, x, i, w: l.forward(x.cpu()),
    "forward_few": lambda l, x, i, w: l.forward_few(x),
    "forward_few, the caller's routing": lambda l, x, i, w: l.forward_few(x, i, w),
    "forward_routed": lambda l, x, i, w: l.forward_routed(x, i, w),
    "forward_noalloc": lambda l, x, i, w: nm._check(_lib.lib().nomas_moe_forward_noalloc(l._h, None, None, 0, None)),
}


@pytest.mark.parametrize("call", NOTHING)
def test_a_forward_without_rows_after_the_callers_routing(call):
    layer, x, _, _ = case(6, 64, 4, 2, 96, "bf16", 1)
    idx, w = torch.zeros(6, 2, dtype=torch.int32, device="cuda"), torch.ones(6, 2, device="cuda")
    layer.forward_few(x, idx, w)
    with pytest.raises(nm.NomasError, match="caller's routing"):
        layer.routing(6)
    NOTHING[call](layer, x[:0], idx[:0], w[:0])
    idx, w, counts, gap = layer.routing(0)
    assert idx.shape == (0, 2) and not counts.any()
