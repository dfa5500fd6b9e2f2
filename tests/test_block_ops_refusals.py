"""What the routing, the routed experts and the block seams refuse -- CPU only.

Through the C ABI: every refusal is decided on the host, before the GPU is
touched.  Through the Python mirror: before the library is called."""
import ctypes as C

import pytest
import torch

import nomas_moe as nm
from nomas_moe import _lib

P = 4096  # an aligned address that nothing reads


def lib():
    return _lib.lib()


def route(dtype=0, logits=P, rows=4, experts=8, top_k=2, scoring=0, bias=None, groups=1, top_groups=1,
          group_top=2, renormalize=1, scale=1.0, eps=1e-9, idx=P, w=P, counts=None):
    return lib().nomas_route(dtype, logits, rows, experts, top_k, scoring, bias, groups, top_groups, group_top,
                             renormalize, scale, eps, idx, w, counts, None)


@pytest.mark.parametrize("code,kw,text", [
    (2, dict(dtype=3), "dtype"), (2, dict(dtype=-1), "dtype"),
    (1, dict(experts=0), "top_k/experts"), (1, dict(top_k=0), "top_k"), (1, dict(top_k=9), "top_k"),
    (1, dict(experts=1025), "maximum"), (2, dict(rows=-1), "rows"), (2, dict(rows=1 << 31), "rows"),
    (1, dict(scoring=2), "scoring"), (2, dict(scale=float("inf")), "scale"), (2, dict(scale=float("nan")), "scale"),
    (2, dict(eps=-1.0), "eps"), (2, dict(eps=float("nan")), "eps"), (2, dict(eps=float("inf")), "eps"),
    (1, dict(groups=0), "groups"), (1, dict(groups=3), "groups"), (1, dict(experts=130, groups=65), "groups"),
    (1, dict(groups=4, top_groups=5), "top_groups"), (1, dict(groups=4, top_groups=0), "top_groups"),
    (1, dict(groups=8, top_groups=1), "do not hold"), (1, dict(groups=2, top_groups=1, group_top=3), "group_top"),
    (2, dict(logits=None), "non-null"), (2, dict(idx=None), "non-null"), (2, dict(w=None), "non-null"),
    (2, dict(logits=P + 2), "misaligned"), (2, dict(dtype=1, logits=P + 1), "misaligned"),
    (2, dict(bias=P + 2), "misaligned"), (2, dict(idx=P + 1), "misaligned"), (2, dict(counts=P + 2), "misaligned"),
])
def test_route(code, kw, text):
    assert route(**kw) == code
    assert text in _lib.last_error()


def test_route_without_rows_is_done():
    assert route(rows=0, logits=None, idx=None, w=None) == 0


@pytest.mark.parametrize("code,kw,text", [
    (2, dict(dtype=7), "dtype"), (1, dict(k=9), "top_k"), (1, dict(scoring=-1), "scoring"),
    (2, dict(logits=None), "non-null"), (2, dict(dw=None), "non-null"), (2, dict(dl=None), "non-null"),
    (2, dict(idx=P + 2), "misaligned"), (2, dict(dl=P + 2), "misaligned"), (2, dict(rows=-3), "rows"),
    (2, dict(eps=-1e-9), "eps"),
])
def test_route_backward(code, kw, text):
    a = dict(dtype=0, logits=P, idx=P, dw=P, rows=4, experts=8, k=2, scoring=0, renorm=1, scale=1.0, eps=1e-9, dl=P)
    a.update(kw)
    assert lib().nomas_route_backward(*a.values(), None) == code
    assert text in _lib.last_error()


SEAM = dict(dtype=1, x=P, y=P, out=P, h=2 * P, rows=6, dim=64, seq=3, gate=None, post=0, post_w=None, alpha=1.0,
            norm_w=None, shift=None, scale=None, eps=1e-6)


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=3), "dtype"), (dict(rows=-1), "rows"), (dict(rows=(1 << 30) + 8, seq=8), "rows"),
    (dict(dim=0), "dim"), (dict(dim=60), "dim"), (dict(dim=16392), "dim"), (dict(seq=0), "seq"),
    (dict(seq=4), "seq"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(alpha=float("inf")), "residual_scale"), (dict(x=None), "non-null"), (dict(y=None), "non-null"),
    (dict(out=None), "non-null"), (dict(h=P), "different"), (dict(x=P + 8), "16-byte"), (dict(h=P + 8), "16-byte"),
    (dict(gate=P + 4), "16-byte"), (dict(shift=P + 4), "16-byte"), (dict(norm_w=P + 8), "16-byte"),
])
def test_block_seam(kw, text):
    assert lib().nomas_block_seam(*{**SEAM, **kw}.values(), None) == 2
    assert text in _lib.last_error()


def test_block_seam_without_rows_is_done():
    assert lib().nomas_block_seam(*{**SEAM, "rows": 0, "x": None, "y": None, "out": None, "h": None}.values(),
                                  None) == 0


BACK = dict(dtype=1, dout=P, dh=P, out=P, y=P, dx=P, dy=2 * P, rows=6, dim=64, seq=3, gate=None, post=1, post_w=None,
            alpha=1.0, norm_w=None, scale=None, eps=1e-6, dgate=P, dshift=P, dscale=P, dnorm_w=P, dpost_w=P,
            workspace=P, nbytes=1 << 40)


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=-1), "dtype"), (dict(dim=20), "dim"), (dict(seq=5), "seq"), (dict(alpha=float("nan")), "residual"),
    (dict(dout=None, dh=None, dshift=None, dscale=None, dnorm_w=None), "dout and dh"), (dict(out=None), "needs out"),
    (dict(y=None), "need y"), (dict(dh=None), "need dh"), (dict(post=0), "post_norm"), (dict(dy=P), "different"),
    (dict(dgate=P + 8), "16-byte"), (dict(dx=P + 2), "16-byte"), (dict(workspace=P + 8), "16-byte"),
    (dict(workspace=None), "workspace"), (dict(nbytes=16), "workspace"), (dict(nbytes=-1), "workspace"),
])
def test_block_seam_backward(kw, text):
    assert lib().nomas_block_seam_backward(*{**BACK, **kw}.values(), None) == 2
    assert text in _lib.last_error()


def test_block_seam_workspace():
    ws = lib().nomas_block_seam_workspace
    assert ws(6, 64, 3) > 0 and ws(14232, 2048, 4744) > 0
    for bad in ((0, 64, 1), (6, 64, 4), (6, 0, 3), (6, 64, 0), (-6, 64, 3), (6, 16392, 3), ((1 << 30) + 8, 64, 8)):
        assert ws(*bad) == 0


def test_forward_routed_needs_a_handle():
    assert lib().nomas_moe_forward_routed(None, P, P, P, P, 4, None) == 2
    assert "handle" in _lib.last_error()


# ---- the Python mirror ----------------------------------------------------------

class _NoLib:
    def __getattr__(self, name):
        raise AssertionError(f"library called: {name}")


@pytest.fixture
def no_lib(monkeypatch):
    monkeypatch.setattr(_lib, "lib", lambda: _NoLib())


def refused(text, f, *a, **kw):
    with pytest.raises(nm.NomasError, match=text):
        f(*a, **kw)


class _Cuda(torch.Tensor):
    """A host tensor that says it is on the GPU, for the checks that come after that one."""
    is_cuda = True


def fake(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype).as_subclass(_Cuda)


def test_mirror_of_route(no_lib):
    refused("device tensors", nm.route, torch.zeros(4, 8), 2)
    refused("device tensors", nm.route_backward, torch.zeros(4, 8), torch.zeros(4, 2), torch.zeros(4, 2))
    refused("f32, bf16 or f16", nm.route, fake(4, 8, dtype=torch.float64), 2)
    refused("scoring", nm.route, fake(4, 8), 2, scoring="tanh")
    refused("top_k", nm.route, fake(4, 8), 9)
    refused("top_k", nm.route, fake(4, 8), 0)
    refused("bias", nm.route, fake(4, 8), 2, bias=torch.zeros(7))
    i, w = fake(4, 2, dtype=torch.int32), fake(4, 2)
    refused("idx", nm.route_backward, fake(4, 8), fake(4, 2, dtype=torch.int64), w)
    refused("idx", nm.route_backward, fake(4, 8), fake(3, 2, dtype=torch.int32), w)
    refused("dw", nm.route_backward, fake(4, 8), i, fake(4, 3))
    refused("dw", nm.route_backward, fake(4, 8), i, fake(4, 2, dtype=torch.bfloat16))


def test_mirror_of_the_seam(no_lib):
    x = fake(2, 3, 16)
    refused("device tensors", nm.block_seam, torch.zeros(2, 3, 16), torch.zeros(2, 3, 16))
    refused("B, L, D", nm.block_seam, fake(3, 16), fake(3, 16))
    refused("^y", nm.block_seam, x, fake(2, 3, 8))
    refused("^y", nm.block_seam, x, fake(2, 3, 16, dtype=torch.bfloat16))
    refused("gate", nm.block_seam, x, x, fake(3, 16))
    refused("scale", nm.block_seam, x, x, None, None, fake(2, 8))
    refused("norm_w", nm.block_seam, x, x, norm_w=fake(15))
    refused("post_norm", nm.block_seam, x, x, post_w=fake(16))
    refused("norm=True", nm.block_seam, x, x, norm=False, shift=fake(2, 16))
    refused("out", nm.block_seam, x, x, out=fake(2, 3, 8))
    refused("^h", nm.block_seam, x, x, out=fake(2, 3, 16), h=fake(2, 4, 16))
    back = nm.block_seam_backward
    refused("dout and dh", back, None, None, x, x)
    refused("needs out", back, None, x, None, x)
    refused("needs y", back, x, x, x, None, post_norm=True)
    refused("gate needs y", back, x, x, x, None, fake(2, 16))
    refused("need dh", back, x, None, None, x, None, fake(2, 16))
    refused("post_norm", back, x, x, x, x, post_w=fake(16))
    refused("dh", back, x, fake(2, 3, 8), x, x)
    refused("^out", back, x, x, fake(1, 3, 16), x)


def test_mirror_of_forward_routed(no_lib):
    layer = object.__new__(nm.MoeLayer)
    layer._h, layer.dim, layer.top_k, layer.dtype, layer.device = None, 16, 2, nm.DataType.F32, 0
    x, i, w = torch.zeros(4, 16), torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2)
    refused("last dim", layer.forward_routed, torch.zeros(4, 8), i, w)
    refused("dtype", layer.forward_routed, x.bfloat16(), i, w)
    refused("GPU", layer.forward_routed, x, i, w)
