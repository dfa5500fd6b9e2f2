"""8-bit values with block scales in 64 bits, for their tests."""
from __future__ import annotations

import torch

BLOCK = 128
LEAST = 2.0 ** -126
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}
F32 = 2.0 ** -24

_codes = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
_middles = (_codes[1:] + _codes[:-1]) / 2


def nearest(v):
    """The nearest e4m3 values of f64 ones in [-448, 448], ties to the even code."""
    size = v.abs()
    lo, hi = torch.searchsorted(_middles, size), torch.searchsorted(_middles, size, right=True)
    return torch.copysign(_codes[torch.where(hi % 2 == 0, hi, lo)], v)


def expand(scale, rows, cols, square):
    s = scale.repeat_interleave(BLOCK, 1)[:, :cols]
    return s.repeat_interleave(BLOCK, 0)[:rows] if square else s


def quantize(x, square):
    """(values, scales) in f64 of a finite f64 matrix; the scales are f32 numbers."""
    rows, cols = x.shape
    rb, kb = -(-rows // BLOCK), -(-cols // BLOCK)
    scale = torch.zeros(rb if square else rows, kb, dtype=torch.float64)
    for i in range(scale.shape[0]):
        for j in range(kb):
            r = slice(i * BLOCK, (i + 1) * BLOCK) if square else slice(i, i + 1)
            scale[i, j] = x[r, j * BLOCK:(j + 1) * BLOCK].abs().max()
    scale = (scale / 448).clamp(min=LEAST).float().double()
    return nearest(x / expand(scale, rows, cols, square)), scale


def product(a, sa, b, sb):
    """(a b^T, the sums of its terms' magnitudes) in f64."""
    x = a.double() * expand(sa.double(), *a.shape, False)
    w = b.double() * expand(sb.double(), *b.shape, True)
    return x @ w.T, x.abs() @ w.abs().T


def product_bound(want, mag, K, dtype):
    """f32 results: a block's 128 products are exact; adding them rounds at most 128 times, by at
    most a step (the matrix cores may truncate), each of the magnitudes' sum; then the scales'
    product, one fused step per block and the sums of up to 8 waves, and the bias; then half a
    step of the output's type.  For 16-bit results the 8-bit instructions drop, of each 8 products,
    what 7 of them have below 2^-13 of the largest one's power of two: 7 x 2^-13 of the
    magnitudes' sum at most."""
    e = (2 * BLOCK + -(-K // BLOCK) + 16) * F32 * mag
    if dtype != torch.float32:
        e = e + 7 * 2.0 ** -13 * mag
    return e + HALF[dtype] * (want.abs() + e) + TINY[dtype]


def random_pair(M, N, K, seed, spread=1.0):
    """(a, sa, b, sb) with scales of different sizes, on the CPU."""
    g = torch.Generator().manual_seed(seed)

    def one(rows, square):
        q = nearest((torch.randn(rows, K, generator=g, dtype=torch.float64) * 100).clamp(-448, 448))
        n = -(-rows // BLOCK) if square else rows
        s = torch.exp(spread * torch.randn(n, -(-K // BLOCK), generator=g)) / 100
        return q.float().to(torch.float8_e4m3fn), s

    return one(M, False) + one(N, True)
