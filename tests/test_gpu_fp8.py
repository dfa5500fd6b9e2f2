"""8-bit quantisation and products with block scales against their definitions in 64 bits."""
import pytest
import torch

import nomas_moe as nm
import _fp8 as F

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def check_quantized(x, square, q, s):
    want, scale = F.quantize(x.double().reshape(-1, x.shape[-1]), square)
    assert q.dtype == nm.FP8 and s.dtype == torch.float32
    assert torch.equal(s.cpu().double().reshape(scale.shape), scale)
    assert torch.equal(q.cpu().double().reshape(want.shape), want)


@pytest.mark.parametrize("square", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 16), (3, 128), (5, 144), (127, 256), (129, 1008), (300, 2064), (1, 8192)])
def test_quantize(rows, cols, dtype, square):
    g = torch.Generator().manual_seed(rows * 31 + cols)
    x = (torch.randn(rows, cols, generator=g) * torch.exp(torch.randn(rows, 1, generator=g))).to(dtype)
    check_quantized(x, square, *nm.quantize_fp8(x.cuda(), square=square))


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_rounds_once(dtype):
    """Quotients next to the middle of two e4m3, where rounding to f32 first would decide otherwise."""
    n = torch.arange(1, 257, dtype=torch.float64)
    x = torch.cat([torch.stack([n, torch.full_like(n, m)]).T.reshape(-1) for m in (201.0, 223.0, 249.0, 255.0)])
    x = x.reshape(-1, 128)
    x = torch.cat([x, -x.flip(1), x * 2.0 ** -10, x / 4]).to(dtype)
    check_quantized(x, False, *nm.quantize_fp8(x.cuda()))


def test_quantize_all_ranges_of_f32():
    g = torch.Generator().manual_seed(5)
    x = torch.randn(64, 128, generator=g)
    e = torch.arange(64)[:, None] * 4 - 126  # rows from 2^-126 to 2^126
    x = torch.ldexp(x.double(), e).float()
    x = torch.cat([x, torch.zeros(1, 128), torch.full((1, 128), 3.0e38), torch.full((1, 128), -2.0 ** -149)])
    check_quantized(x, False, *nm.quantize_fp8(x.cuda()))


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("square", [False, True])
def test_quantize_what_is_not_finite(bad, square):
    x = torch.randn(200, 400, generator=torch.Generator().manual_seed(1))
    want, scale = F.quantize(x.double(), square)
    x[150, 300] = bad
    q, s = nm.quantize_fp8(x.cuda(), square=square)
    r = slice(128, 200) if square else slice(150, 151)
    want[r, 256:384] = float("nan")
    scale[1 if square else 150, 2] = float("nan")
    assert torch.equal(q.cpu().double().nan_to_num(999), want.nan_to_num(999))
    assert torch.equal(s.cpu().double().nan_to_num(999), scale.nan_to_num(999))


def test_quantize_shapes_strides_and_nothing():
    x = torch.randn(3, 5, 64, device="cuda")
    q, s = nm.quantize_fp8(x)
    assert q.shape == (3, 5, 64) and s.shape == (3, 5, 1)
    check_quantized(x.cpu(), False, q, s)
    t = torch.randn(64, 7, device="cuda").T
    check_quantized(t.cpu().contiguous(), False, *nm.quantize_fp8(t))
    q, s = nm.quantize_fp8(torch.zeros(0, 32, device="cuda"))
    assert q.shape == (0, 32) and s.shape == (0, 1)
    q, s = nm.quantize_fp8(torch.zeros(0, 32, device="cuda"), square=True)
    assert q.shape == (0, 32) and s.shape == (0, 1)
    q, s = nm.quantize_fp8(torch.randn(32, device="cuda"))
    assert q.shape == (32,) and s.shape == (1,)


# from one row to the sizes that take each of the kernels
SIZES = [(1, 1, 16), (1, 40, 128), (3, 130, 272), (16, 64, 1024), (17, 129, 400), (32, 96, 640), (33, 257, 144),
         (64, 512, 2048), (200, 321, 1008), (512, 64, 128), (600, 515, 272), (1111, 2667, 1008), (4100, 3077, 144),
         (3333, 4096, 400), (3333, 4099, 400), (1, 8200, 272), (5, 16400, 144), (20, 8200, 144), (20, 16400, 144),
         (128, 8192, 1024), (256, 2048, 1024)]


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", SIZES)
def test_matmul(M, N, K, dtype, bias):
    a, sa, b, sb = F.random_pair(M, N, K, M + N + K)
    want, mag = F.product(a, sa, b, sb)
    c = torch.randn(N, generator=torch.Generator().manual_seed(2)) if bias else None
    if bias:
        want, mag = want + c.double(), mag + c.double().abs()
    # the operands and the result inside of larger buffers: what stands behind them is not used, nor written
    def inside(t):
        n = t.numel()
        big = torch.full((n + 4096,), float("nan"), device="cuda", dtype=torch.float32).to(t.dtype)
        big[2048:2048 + n] = t.reshape(-1).cuda()
        return big[2048:2048 + n].view(t.shape)
    out = torch.full((M * N + 64,), 7.0, dtype=dtype, device="cuda")
    y = nm.matmul_fp8(inside(a), inside(sa), inside(b), inside(sb), None if c is None else c.cuda(), dtype=dtype,
                      out=out[:M * N].view(M, N))
    assert bool((out[M * N:] == 7.0).all())
    off = (y.cpu().double() - want).abs() - F.product_bound(want, mag, K, dtype)
    assert float(off.max()) <= 0.0


@pytest.mark.parametrize("M", [3, 40, 700])
def test_matmul_keeps_rows_apart(M):
    """A NaN value, an infinite and a zero scale reach their own rows and columns only."""
    N, K = 300, 400
    a, sa, b, sb = F.random_pair(M, N, K, 9)
    sa[0, 0], sa[1, 3] = float("inf"), 0.0
    bits = a.view(torch.uint8)
    bits[2, 399] = 0x7f
    sb[2, 1] = float("nan")
    sa2 = sa.clone()
    sa2[0, 0] = 1.0
    a2 = a.clone()
    a2.view(torch.uint8)[2, 399] = 0
    sb2 = sb.clone()
    sb2[2, 1] = 1.0
    want, mag = F.product(a2, sa2, b, sb2)
    y = nm.matmul_fp8(a.cuda(), sa.cuda(), b.cuda(), sb.cuda(), dtype=torch.float32).cpu().double()
    assert bool(y[2].isnan().all()) and not bool(y[0, :256].isfinite().any()) and bool(y[:, 256:].isnan().all())
    keep = torch.arange(M) != 0
    keep[2] = False
    off = (y - want).abs() - F.product_bound(want, mag, K, torch.float32)
    assert float(off[keep][:, :256].max()) <= 0.0


def test_matmul_leading_dimensions_strides_and_nothing():
    a, sa, b, sb = (t.cuda() for t in F.random_pair(6, 40, 256, 3))
    y = nm.matmul_fp8(a, sa, b, sb)
    assert torch.equal(nm.matmul_fp8(a.view(2, 3, 256), sa.view(2, 3, 2), b, sb), y.view(2, 3, 40))
    assert torch.equal(nm.matmul_fp8(a[0], sa[0], b, sb), y[0])
    wide = torch.zeros(6, 512, device="cuda").to(nm.FP8)
    wide[:, 128:384] = a
    assert torch.equal(nm.matmul_fp8(wide[:, 128:384], sa, b, sb), y)
    assert torch.equal(nm.matmul_fp8(a, sa.T.contiguous().T, b, sb), y)
    assert nm.matmul_fp8(a[:0], sa[:0], b, sb).shape == (0, 40)
    assert nm.matmul_fp8(a, sa, b[:0], sb[:0]).shape == (6, 0)
    with pytest.raises(nm.NomasError, match="misaligned"):
        nm.matmul_fp8(a.view(-1)[8:264].view(1, 256), sa[:1], b, sb)


def test_quantize_then_matmul():
    """Used together: the product of the quantised operands is the product of their values."""
    x = torch.randn(37, 784, device="cuda", dtype=torch.bfloat16)
    w = torch.randn(210, 784, device="cuda", dtype=torch.bfloat16)
    a, b = nm.quantize_fp8(x), nm.quantize_fp8(w, square=True)
    y = nm.matmul_fp8(*a, *b, dtype=torch.float32)
    (qa, sa), (qb, sb) = F.quantize(x.cpu().double(), False), F.quantize(w.cpu().double(), True)
    want, mag = F.product(qa, sa, qb, sb)
    assert bool(((y.cpu().double() - want).abs() <= F.product_bound(want, mag, 784, torch.float32)).all())
    # each value is off by at most half a step of e4m3, 2^-4 of it (or of the smallest normal value, 2^-6)
    for t, (q, s), sq in ((x, (qa, sa), False), (w, (qb, sb), True)):
        v, e = t.cpu().double(), F.expand(s, *t.shape, sq)
        assert bool(((q * e - v).abs() <= 2.0 ** -4 * (1 + 2.0 ** -20) * torch.maximum(v.abs(), e * 2.0 ** -6)).all())


@pytest.mark.parametrize("M", [5, 700])
def test_streams_and_capture(M):
    a, sa, b, sb = (t.cuda() for t in F.random_pair(M, 520, 656, 4))
    x = torch.randn(M, 656, device="cuda")
    want, (wq, ws) = nm.matmul_fp8(a, sa, b, sb), nm.quantize_fp8(x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y, (q, c) = nm.matmul_fp8(a, sa, b, sb), nm.quantize_fp8(x)
    s.synchronize()
    assert torch.equal(y, want) and torch.equal(q.view(torch.uint8), wq.view(torch.uint8)) and torch.equal(c, ws)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        q, c = nm.quantize_fp8(x)
        y = nm.matmul_fp8(q, c, b, sb)
    for seed in range(3):
        x.copy_(torch.randn(M, 656, generator=torch.Generator().manual_seed(seed)))
        eager = nm.matmul_fp8(*nm.quantize_fp8(x), b, sb)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, eager)
