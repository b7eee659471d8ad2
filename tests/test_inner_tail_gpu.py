"""A reduction that ends inside 16 bytes of a wider, aligned pitch: what lies behind it in the buffers, infinities and NaN
included, never enters a product."""
import ctypes as C

import pytest
import torch

from beantensor_b200 import _lib
from tests import ragged

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def spoilt(shape, inner, dtype, seed):
    """Normal values in the first `inner` columns of a buffer whose other columns are infinities and NaN."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(shape, generator=g, device="cuda").to(dtype)
    x[..., inner:] = float("nan")
    x[..., inner::2] = float("inf")
    return x[..., :inner]


@pytest.mark.parametrize("kernel", ["1cta", "2cta", "decode"])
@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("K", [1, 7, 33, 65, 66, 67, 191, 577])
def test_grouped_product(btm, monkeypatch, kernel, trans, K):
    monkeypatch.setenv("BTM_FORCE_KERNEL", kernel)
    bounds, rows, N, pitch = [0, 50, 50, 190], 200, 136, (K + 7) // 8 * 8
    t = torch.tensor(bounds, dtype=torch.int32, device="cuda")
    a = spoilt((rows, pitch), K, BF16, 1)
    b = spoilt((3, N, pitch), K, BF16, 2).transpose(1, 2) if trans else spoilt((3, K, N), N, BF16, 2)
    out = torch.zeros((rows, N), dtype=BF16, device="cuda")
    btm.grouped_matmul_gpu(a, b, t, out)
    btm.check_device_status(0)
    for g, (lo, hi) in enumerate(ragged.spans(bounds, rows)):
        if hi > lo:
            ragged.check(out[lo:hi], *ragged.product(a[lo:hi], b[g]), K)
    assert (out[190:] == 0).all()


@pytest.mark.parametrize("M,N", [(65, 33), (7, 130), (1, 1), (130, 133)])
def test_grouped_gradient(btm, M, N):
    # Here the inner extents are the output's: what lies behind them must not reach the columns that are stored.
    bounds, rows = [0, 50, 50, 190], 200
    t = torch.tensor(bounds, dtype=torch.int32, device="cuda")
    a, d = spoilt((rows, (M + 7) // 8 * 8), M, F16, 1), spoilt((rows, (N + 7) // 8 * 8), N, F16, 2)
    out = torch.full((3, M, N), 5.0, dtype=F16, device="cuda")
    btm.grouped_matmul_wgrad_gpu(a, d, t, out)
    btm.check_device_status(0)
    for g, (lo, hi) in enumerate(ragged.spans(bounds, rows)):
        ragged.check(out[g], *ragged.product(a[lo:hi].t(), d[lo:hi]), hi - lo)


@pytest.mark.parametrize("kernel", ["1cta", "2cta"])
@pytest.mark.parametrize("K", [1, 7, 33, 65, 66, 67, 191, 577])
def test_dense_product(btm, monkeypatch, kernel, K):
    monkeypatch.setenv("BTM_FORCE_KERNEL", kernel)
    M, N, pitch = 150, 136, (K + 7) // 8 * 8
    a, b = spoilt((M, pitch), K, F16, 1), spoilt((K, N), N, F16, 2)
    out = torch.empty((M, N), dtype=F16, device="cuda")
    btm.matmul_gpu(a, b, out)
    btm.check_device_status(0)
    ragged.check(out, *ragged.product(a, b), K)
    bt = spoilt((N, pitch), K, F16, 3)
    st = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert _lib.lib().btm_gemm_bt(0, st, _lib.F16, M, N, K, a.data_ptr(), pitch, bt.data_ptr(), pitch, out.data_ptr(), N) == _lib.OK
    btm.check_device_status(0)
    ragged.check(out, *ragged.product(a, bt.t()), K)
