"""8-bit products whose scales' products leave f32's range while the results do not.

Bounds as in _fp8.product_bound: it counts one rounding for the scales' product and one a block; with the
scales' powers of two applied apart there is one more for the whole sum, within its 16 spare ones.
"""
import pytest
import torch

import nomas_moe as nm
import _fp8 as F
from test_gpu_ffn_fp8 import case, layer_of, wanted

pytestmark = pytest.mark.gpu

# one size for each of the kernels (rows, columns, tiles of 128 and of 256), ragged ones
SIZES = [(1, 40, 272), (3, 130, 1296), (20, 96, 640), (20, 8200, 272), (20, 16400, 144), (64, 512, 2048), (200, 321, 1008),
         (1111, 2667, 272), (3333, 4096, 400), (3333, 4099, 400)]


def scales(n, kb, e, g):
    """2^e times numbers between 1/2 and 3/2, of either sign."""
    s = torch.ldexp(2 * torch.rand(n, kb, generator=g, dtype=torch.float64) - 1 + 1e-3, torch.tensor(e))
    return torch.where(s >= 0, s + 2.0 ** (e - 1), s - 2.0 ** (e - 1)).float()


def run(a, sa, b, sb, dtype, bias=None, more=0.0):
    want, mag = F.product(a, sa, b, sb)
    if bias is not None:
        want, mag = want + bias.double(), mag + bias.double().abs()
    y = nm.matmul_fp8(a.cuda(), sa.cuda(), b.cuda(), sb.cuda(), None if bias is None else bias.cuda(), dtype=dtype)
    off = (y.cpu().double() - want).abs() - F.product_bound(want, mag, a.shape[1], dtype) - more
    assert float(off.max()) <= 0.0
    return want


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_products_of_scales_below_the_smallest_normal(M, N, K, dtype):
    """Rows of 1e-36, as the quantiser scales them, by weights of 1e-2; and scales whose product f32 does not hold at all."""
    g = torch.Generator().manual_seed(M + N)
    a, _, b, _ = F.random_pair(M, N, K, M + N + K)
    kb, nb = -(-K // 128), -(-N // 128)
    want = run(a, scales(M, kb, -125, g), b, scales(nb, kb, -14, g), dtype)
    assert float(want.abs().max()) > 2.0 ** -126
    # results below the smallest normal: the sums of up to eight waves and their total are at f32's last bit
    run(a, scales(M, kb, -125, g), b, scales(nb, kb, -26, g), dtype, more=9 * 2.0 ** -150)
    # (2^-170 and less: nothing is left of a result)
    run(a, scales(M, kb, -110, g), b, scales(nb, kb, -60, g), dtype, more=9 * 2.0 ** -150)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_products_of_scales_above_the_largest(M, N, K, dtype):
    g = torch.Generator().manual_seed(M + N)
    kb, nb = -(-K // 128), -(-N // 128)
    # values of a few times 2^-9: a block's sums are at most 128 x 2^-12
    a, b = ((torch.randint(-7, 8, (n, K), generator=g) * 2.0 ** -9).to(torch.float8_e4m3fn) for n in (M, N))
    want = run(a, scales(M, kb, 70, g), b, scales(nb, kb, 59, g), dtype)
    assert bool(want.isfinite().all()) and float(want.abs().max()) > 2.0 ** 100
    # (the same sums where no product is out of range, from 2^55 on and below)
    for e in (50, 54, 60):
        run(a, scales(M, kb, e - 20, g), b, scales(nb, kb, 20, g), dtype, scales(1, N, e - 10, g)[0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_a_sum_of_zero_stays_zero(M, N, K, dtype):
    """Blocks whose scales multiply to infinity, or one of which is 0, beside others; their sums are 0."""
    a, sa, b, sb = F.random_pair(M, N, K, M + N + K)
    a = a.float()
    a[:, :128] = 0
    a = a.to(torch.float8_e4m3fn)
    sa[:, 0], sb[:, 0] = 2.0 ** 100, 2.0 ** 100
    run(a, sa, b, sb, dtype)
    sa[0, 0], sa[-1, 0], sb[-1, 0] = 0.0, -3.0e38, 3.0e38
    run(a, sa, b, sb, dtype)
    # (a scale of 0 beside one next to the largest, and sums that are not 0)
    a, *_ = F.random_pair(M, N, K, M + N + K)
    sa[:, 0] = 0.0
    run(a, sa, b, sb, dtype)


@pytest.mark.parametrize("M", [3, 40, 700])
def test_scales_that_are_not_finite_keep_to_their_rows(M):
    N, K = 300, 400
    a, sa, b, sb = F.random_pair(M, N, K, 9)
    sa2 = sa.clone()
    sa2[0, 1], sa2[2, 3], sa2[1, 0] = float("inf"), float("nan"), 2.0 ** 126
    sb2 = sb.clone()
    sb2[2, 1] = float("-inf")
    want, mag = F.product(a, sa2, b, sb2)
    y = nm.matmul_fp8(a.cuda(), sa2.cuda(), b.cuda(), sb2.cuda(), dtype=torch.float32).cpu().double()
    assert bool(y[2].isnan().all()) and not bool(y[0].isfinite().any()) and not bool(y[:, 256:].isfinite().any())
    keep = torch.arange(M) != 0
    keep[2] = False
    fits = want[keep][:, :256].abs() < 2.0 ** 127
    off = (y - want).abs() - F.product_bound(want, mag, K, torch.float32)
    assert bool((off[keep][:, :256][fits] <= 0.0).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16])
@pytest.mark.parametrize("rows,D,H", [(5, 256, 384), (24, 256, 300), (64, 384, 128), (300, 256, 384), (3100, 256, 2304)])
def test_feed_forward(rows, D, H, dtype):
    """A column of 2^102 beside weights of zero, and weights of 2^42 beside values of zero."""
    x, w, b = case(rows, D, H, rows + D + H)
    x[:, :128] = 0
    x[:, 0] = 7 * 2.0 ** 100
    for n in ("gate", "up"):
        w[n][:, :128] = 0
        w[n][:, 1] = 7 * 2.0 ** 40
    layer = layer_of(w, b, dtype)
    y = layer.forward_fp8(x.to(dtype).cuda())
    want, off = wanted(x, w, b, dtype)
    assert bool(((y.cpu().double() - want).abs() <= off).all())
