"""What the 8-bit quantiser and product refuse -- CPU only (decided on the host)."""
import pytest
import torch

import nomas_moe as nm
from nomas_moe import _lib

P = 1 << 20  # aligned addresses that nothing reads, far apart
STEP = 1 << 24

QUANT = dict(dtype=1, x=P, rows=6, cols=64, square=0, q=P + STEP, scale=P + 2 * STEP)


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(cols=0), "cols"), (dict(cols=24), "cols"),
    (dict(cols=-16), "cols"), (dict(cols=1 << 31), "cols"), (dict(rows=-1), "rows"), (dict(rows=1 << 31), "rows"),
    (dict(rows=1 << 30, cols=512), "rows"), (dict(rows=65536 * 128, square=1), "rows"),
    (dict(x=None), "non-null"), (dict(q=None), "non-null"), (dict(scale=None), "non-null"),
    (dict(x=P + 8), "misaligned"), (dict(q=P + STEP + 4), "misaligned"), (dict(scale=P + 2), "misaligned"),
    (dict(q=P), "shares"), (dict(q=P + 6 * 64 * 2 - 16), "shares"), (dict(scale=P + 16), "shares"),
    (dict(scale=P + STEP + 16), "shares"),
])
def test_quantize(kw, text):
    assert _lib.lib().nomas_quantize_fp8(*{**QUANT, **kw}.values(), None) == 2
    assert text in _lib.last_error()


PRODUCT = dict(dtype=1, a=P, a_scale=P + STEP, b=P + 2 * STEP, b_scale=P + 3 * STEP, bias=None, y=P + 4 * STEP, rows=6,
               n=40, k=64)


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=4), "dtype"), (dict(k=0), "k must"), (dict(k=40), "k must"), (dict(k=(1 << 22) + 16), "k must"),
    (dict(n=-1), "n="), (dict(n=(1 << 24) + 1), "n="), (dict(rows=-1), "rows"), (dict(rows=(1 << 30) + 1), "rows"),
    (dict(a=None), "non-null"), (dict(a_scale=None), "non-null"), (dict(b=None), "non-null"),
    (dict(b_scale=None), "non-null"), (dict(y=None), "non-null"), (dict(a=P + 8), "misaligned"),
    (dict(b=P + 1), "misaligned"), (dict(y=P + 4 * STEP + 8), "misaligned"), (dict(a_scale=P + 2), "misaligned"),
    (dict(b_scale=P + 1), "misaligned"), (dict(bias=P + 2), "misaligned"), (dict(y=P), "shares"),
    (dict(y=P + STEP), "shares"), (dict(y=P + 2 * STEP + 16), "shares"), (dict(y=P + 3 * STEP), "shares"),
    (dict(bias=P + 4 * STEP + 4), "shares"), (dict(y=P - 16), "shares"),
])
def test_matmul(kw, text):
    assert _lib.lib().nomas_matmul_fp8(*{**PRODUCT, **kw}.values(), None) == 2
    assert text in _lib.last_error()


def test_nothing_to_do_is_done():
    lib = _lib.lib()
    assert lib.nomas_quantize_fp8(*{**QUANT, "rows": 0, "x": None, "q": None, "scale": None}.values(), None) == 0
    for kw in (dict(rows=0), dict(n=0)):
        assert lib.nomas_matmul_fp8(*{**PRODUCT, **kw, "a": None, "y": None}.values(), None) == 0


# ---- the Python mirror ----------------------------------------------------------

class _NoLib:
    def __getattr__(self, name):
        raise AssertionError(f"library called: {name}")


@pytest.fixture
def no_lib(monkeypatch):
    monkeypatch.setattr(_lib, "lib", lambda: _NoLib())


class _Cuda(torch.Tensor):
    """A host tensor that says it is on the GPU, for the checks that come after that one."""
    is_cuda = True


def fake(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype).as_subclass(_Cuda)


def refused(text, f, *a, **kw):
    with pytest.raises(nm.NomasError, match=text):
        f(*a, **kw)


def test_mirror_of_quantize(no_lib):
    refused("device tensors", nm.quantize_fp8, torch.zeros(4, 64))
    refused("f32, bf16 or f16", nm.quantize_fp8, fake(4, 64, dtype=torch.float64))
    refused("multiple of 16", nm.quantize_fp8, fake(4, 40))
    refused("multiple of 16", nm.quantize_fp8, fake(4, 0))
    refused("shape", nm.quantize_fp8, fake(2, 4, 64), square=True)
    refused("shape", nm.quantize_fp8, torch.zeros(()).as_subclass(_Cuda))


def test_mirror_of_matmul(no_lib):
    f8 = nm.FP8
    a, b, sa, sb = fake(6, 144, dtype=f8), fake(40, 144, dtype=f8), fake(6, 2), fake(1, 2)
    mm = nm.matmul_fp8
    refused("one GPU", mm, torch.zeros(6, 144).to(f8), sa, b, sb)
    refused("must be", mm, fake(6, 144), sa, b, sb)
    refused("values", mm, a, sa, fake(40, 128, dtype=f8), sb)
    refused("values", mm, a, sa, fake(2, 40, 144, dtype=f8), sb)
    refused("multiple of 16", mm, fake(6, 24, dtype=f8), fake(6, 1), fake(40, 24, dtype=f8), fake(1, 1))
    refused("a_scale", mm, a, fake(6, 1), b, sb)
    refused("a_scale", mm, a, fake(6, 2, dtype=torch.bfloat16), b, sb)
    refused("b_scale", mm, a, sa, b, fake(2, 2))
    refused("bias", mm, a, sa, b, sb, fake(41))
    refused("result", mm, a, sa, b, sb, dtype=torch.float64)
    refused("out", mm, a, sa, b, sb, out=fake(6, 41, dtype=torch.bfloat16))
    refused("out", mm, a, sa, b, sb, out=fake(6, 40))
    refused("contiguous", mm, a, sa, b, sb, out=fake(40, 6, dtype=torch.bfloat16).T)


# ---- the layers -------------------------------------------------------------------

def test_layers_need_a_handle():
    lib = _lib.lib()
    for call in (lambda: lib.nomas_moe_forward_few(None, P, None, None, 0, P, 4, None), lambda: lib.nomas_moe_quantize(None),
                 lambda: lib.nomas_ffn_quantize(None), lambda: lib.nomas_ffn_forward_fp8(None, P, P, 4, None)):
        assert call() == 2
        assert "handle" in _lib.last_error()


def test_mirror_of_the_layers(no_lib):
    layer = object.__new__(nm.MoeLayer)
    layer._h, layer.dim, layer.top_k, layer.dtype, layer.device = None, 16, 2, nm.DataType.F32, 0
    x, i, w = torch.zeros(4, 16), torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2)
    refused("last dim", layer.forward_few, torch.zeros(4, 8))
    refused("dtype", layer.forward_few, x.bfloat16())
    refused("GPU", layer.forward_few, x)
    refused("GPU", layer.forward_few, x, i, w)
    ffn = object.__new__(nm.FeedForward)
    ffn._h, ffn.dim, ffn.dtype, ffn.device = None, 16, nm.DataType.F32, 0
    refused("last dim", ffn.forward_fp8, torch.zeros(4, 8))
    refused("dtype", ffn.forward_fp8, x.bfloat16())
    refused("GPU", ffn.forward_fp8, x)


def test_quantize_refuses_more_blocks_than_a_grid_holds():
    kw = dict(rows=1 << 30, cols=16, q=P + (1 << 40), scale=P + (1 << 41))
    assert _lib.lib().nomas_quantize_fp8(*{**QUANT, **kw}.values(), None) == 2
    assert "rows" in _lib.last_error()
