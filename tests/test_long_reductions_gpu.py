"""Reductions so long that a tile alone takes more than the bounded waits' base limit: a wait for work that goes on is no hang. The
limit is lowered instead of the reduction made a thousand times longer."""
import pytest
import torch

from beantensor_b200 import _lib
from tests import ragged

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
LENGTH = 2_000_000


@pytest.fixture
def short_limit(btm):
    btm.check_device_status(0)
    L = _lib.lib()
    assert L.btm_debug_set(b"wait_limit_cycles", 200_000) == _lib.OK
    yield
    assert L.btm_debug_set(b"wait_limit_cycles", 0) == _lib.OK


def signs(shape, seed):
    """-1, 0 and 1: no partial sum leaves the whole numbers below 2^24, so that fp32 accumulation is exact."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-1, 2, shape, generator=g, device="cuda").to(BF16)


def test_gradient(btm, short_limit):
    a, d = signs((LENGTH, 8), 1), signs((LENGTH, 8), 2)
    out = torch.empty((2, 8, 8), dtype=BF16, device="cuda")
    btm.grouped_matmul_wgrad_gpu(a, d, torch.tensor([0, 100, LENGTH], dtype=torch.int32, device="cuda"), out)
    btm.check_device_status(0)
    for g, (lo, hi) in enumerate(((0, 100), (100, LENGTH))):
        ragged.check(out[g], *ragged.product(a[lo:hi].t(), d[lo:hi]), 0)


@pytest.mark.parametrize("kernel", ["1cta", "2cta", "decode"])
def test_grouped_product(btm, short_limit, monkeypatch, kernel):
    monkeypatch.setenv("BTM_FORCE_KERNEL", kernel)
    a, b = signs((2, LENGTH), 1), signs((2, LENGTH, 8), 2)
    out = torch.empty((2, 8), dtype=BF16, device="cuda")
    btm.grouped_matmul_gpu(a, b, torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda"), out)
    btm.check_device_status(0)
    for g in range(2):
        ragged.check(out[g:g + 1], *ragged.product(a[g:g + 1], b[g]), 0)


@pytest.mark.parametrize("kernel", ["1cta", "2cta"])
def test_dense_product(btm, short_limit, monkeypatch, kernel):
    monkeypatch.setenv("BTM_FORCE_KERNEL", kernel)
    a, b = signs((8, LENGTH), 1), signs((LENGTH, 8), 2)
    out = torch.empty((8, 8), dtype=BF16, device="cuda")
    btm.matmul_gpu(a, b, out)
    btm.check_device_status(0)
    ragged.check(out, *ragged.product(a, b), 0)


@pytest.mark.parametrize("kernel", ["1cta", "2cta", "decode"])
def test_microscaled_product(btm, short_limit, monkeypatch, kernel):
    monkeypatch.setenv("BTM_FORCE_KERNEL", kernel)
    K = 8 * LENGTH
    x, w = signs((2, K), 1), signs((8, K), 2)
    x[:, ::32], w[:, ::32] = 1, 1  # every block of 32 has a largest value of 1
    xq, wq = torch.empty((2, K // 2), dtype=torch.uint8, device="cuda"), torch.empty((8, K // 2), dtype=torch.uint8, device="cuda")
    xs, ws = (torch.empty(btm.mxfp4_scale_bytes(n, K), dtype=torch.uint8, device="cuda") for n in (2, 8))
    btm.quantize_mxfp4_gpu(x, xq, xs)
    btm.quantize_mxfp4_gpu(w, wq, ws)
    out = torch.empty((2, 8), dtype=BF16, device="cuda")
    btm.matmul_mxfp4_gpu(xq, xs, wq, ws, out)
    btm.check_device_status(0)
    ragged.check(out, *ragged.product(x, w.t()), 0)
