"""8-bit values and products whose tensors pass 4 GiB: the last rows, where 32-bit offsets would wrap,
against the definition in 64 bits.  All else is zero, and has to come out so."""
import pytest
import torch

import nomas_moe as nm
import _fp8 as F

pytestmark = pytest.mark.gpu


def last(whole, part):
    """Zeros with `part` as the last rows, on the device."""
    t = torch.zeros(whole, part.shape[1], dtype=torch.float32 if part.dtype == torch.float32 else torch.uint8, device="cuda")
    t[whole - part.shape[0]:] = part.cuda() if part.dtype == torch.float32 else part.view(torch.uint8).cuda()
    return t if part.dtype == torch.float32 else t.view(nm.FP8)


# outputs; activations, in the kernels of many and of few rows; weights in both
@pytest.mark.parametrize("M,N,K,dtype", [
    (270_000, 8_200, 128, torch.bfloat16), (140_000, 8_200, 144, torch.float32), (600_000, 64, 8_192, torch.bfloat16),
    (600_000, 64, 8_192, torch.float32), (5, 600_064, 8_192, torch.bfloat16), (200, 600_064, 8_192, torch.float16),
    (4_300_000, 8, 1_024, torch.bfloat16),
])
def test_matmul(M, N, K, dtype):
    m, n = min(M, 70), N if N < 10_000 else 256  # (whole blocks of 128 weight rows)
    a, sa, b, sb = F.random_pair(m, n, K, 3)
    want, mag = F.product(a, sa, b, sb)
    y = nm.matmul_fp8(last(M, a), last(M, sa), last(N, b), last(-(-N // 128), sb), dtype=dtype)
    off = (y[M - m:, N - n:].cpu().double() - want).abs() - F.product_bound(want, mag, K, dtype)
    assert float(off.max()) <= 0.0
    assert not bool(y[:M - m].any()) and not bool(y[:, :N - n].any())


def test_quantize():
    g = torch.Generator().manual_seed(1)
    part = torch.randn(130, 8_192, generator=g).to(torch.bfloat16)
    x = torch.zeros(600_000, 8_192, dtype=torch.bfloat16, device="cuda")
    x[-130:] = part.cuda()
    q, s = nm.quantize_fp8(x)
    want, scale = F.quantize(part.double(), False)
    assert torch.equal(q[-130:].cpu().double(), want) and torch.equal(s[-130:].cpu().double(), scale)
    assert not bool(q[:-130].view(torch.uint8).any())
    q, s = nm.quantize_fp8(x, square=True)  # the last square: 600,000 is 128 x 4,687 + 64 rows
    want, scale = F.quantize(part[-64:].double(), True)
    assert torch.equal(q[-64:].cpu().double(), want) and torch.equal(s[-1:].cpu().double(), scale)
