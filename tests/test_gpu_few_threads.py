"""forward_few from two host threads, a layer each."""
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

from test_gpu_few import case

pytestmark = pytest.mark.gpu


def test_two_host_threads():
    # many slots a row, of two numbers: each call's lists need their own share of LDS, past 64 KB with the rest
    layers = [case(64, 40, E, E, 24, "bf16", E)[:2] for E in (64, 128)]

    def call(t):
        return [t[0].forward_few(t[1]).clone() for _ in range(50)]

    want = [layer.forward_few(x) for layer, x in layers]
    torch.cuda.synchronize()
    with ThreadPoolExecutor(2) as pool:
        for _ in range(10):
            got = list(pool.map(call, layers))
            torch.cuda.synchronize()
            assert all(torch.equal(g, w) for gs, w in zip(got, want) for g in gs)
